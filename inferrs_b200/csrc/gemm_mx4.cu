// y[t, f] = sum_k x[t, k] * w[f, k] with w in 4 bits, on the fifth-generation tensor cores (block-scaled products).
//
// The weights are the 128-row operand, the tokens the N dimension, as in gemm_tcgen05.cu; the weights stay 4-bit numbers
// all the way into the tensor core, which multiplies by their powers of two itself.  Two kinds:
//
//   rows that keep their precision   x = s p0 + s/32 p1 + s/32^2 p2 + ..., with s the power of two that puts the largest
//       number of a block of 32 into 128 .. 256, p0 the nearest e4m3 number to x / s and every further one to 32 times what
//       is left.  An e4m3 number has four significant bits, so what is left is at most 2^-4 of a number, and 32 times that
//       fits the same range: every piece adds five bits.  A bfloat16 number is two pieces: p1 holds what p0 leaves of its
//       eight bits exactly, down to 2^-14 of the block's largest number; below, x is off by at most 2^-22 of that.  A float32
//       number is five: off by at most 2^-25 of itself or 2^-37 of the block's largest.  The pieces are columns of one
//       product (kind::mxf8f6f4: w e2m1, x e4m3), whose results are added up at the end, the smallest first.
//   4-bit rows   both operands as they are (kind::mxf4).
//
// TMA brings tiles of 128 weight rows and of tokens into a ring of 128-byte-swizzled stages (4-bit weights beside 8-bit
// pieces are spread to a byte each on the way), and 512-byte tiles of scales, which the issuing thread copies into tensor
// memory in front of the products that use them (every stage has its own columns, so none is overwritten early).
// Accumulators are float32 in tensor memory.  Roles: warp 0 copies (warp 6 the scales, where they are tiles), warp 1 issues
// products, warps 2..5 read back.  Up to four bfloat16 rows are brought to pieces inside the product, by warps 6.. of every CTA while
// the weights stream in; more rows by a kernel of their own.  The product starts while that one runs, but reads weights before the kernels
// ahead have ended only where the library's switch says that none of them writes any.
//
// Up to 64 rows (few_rows_kernel), where low tiles would keep the tensor core longer than the weights take, K is cut over a cluster
// (1, 1, splits): every CTA sends its partial sums to their owners (each has an equal share of the tile's rows) through
// distributed shared memory, one cluster barrier follows, and the owner adds them in the order of the ranks.  More rows
// (gemm_kernel): pairs of CTAs.  Every wait is bounded and reports through this file's error word.
#include <cuda.h>

#include "few_bits.cuh"
#include "sm100.cuh"

namespace mx4 {

using namespace sm100;

constexpr int BM = 128, THREADS = 192, A_BYTES = BM * 128;
// up to so many bfloat16 rows are brought to pieces inside the product (4,096 x 24,576: four rows 13.4 us, eight 16.2 and by themselves 13.3, 13.7 outside
// captured steps)
constexpr int INSIDE_ROWS = 4;
// what a kernel's rows are: the number of pieces of a number, CODES for 4-bit rows
enum { CODES = 1, PIECES_BF16 = 2, PIECES_F32 = 5 };

__device__ int g_error = 0;
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, int code) {
    return mbar_wait_bounded(bar, parity, &g_error, code);
}

struct Params {
    void* y;
    long ldy;
    int y_is_f32, y_wide, n_tok, n_out, num_kb;      // num_kb: stages that K takes
    const unsigned char *w_scales, *x_scales;
    int scale_tiles;                         // 128-column tiles of scales per 128 rows
    const void* x;                           // rows that are brought to pieces inside: ldx elements apart, k numbers each
    long ldx;
    int k, wide;                             // wide: rows start on 16 bytes
    int wait_first;                          // the kernel ahead may have written the weights: nothing is read before it is done
};

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// where CTA `rank` of the cluster has what stands at `local` here
__device__ __forceinline__ unsigned at_rank(unsigned local, unsigned rank) {
    unsigned there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(local), "r"(rank));
    return there;
}
__device__ __forceinline__ void st_remote_f32x4(unsigned there, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// `bytes` (a multiple of 16) from global to shared memory
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Operand descriptors by their low word, which holds where a tile starts in units of 16 bytes: the thread that issues the products
// has about five cycles for an instruction, and what it computes for a stage decides how fast stages follow one another.
__device__ __forceinline__ unsigned long long from_words(unsigned lo, unsigned hi) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
// One lane of the warp, the same every time.  The warp runs the loop around what that lane issues as a whole, so that addresses and
// descriptors stay uniform registers, which the instructions want.
__device__ __forceinline__ bool elected() {
    unsigned r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
constexpr unsigned TILE_HI = (unsigned)(1024 >> 4) | 1u << 14 | 2u << 29, TILE_LO = 1u << 16;       // desc_k_major in sm100.cuh
constexpr unsigned SCALE_HI = (unsigned)(128 >> 4) | 1u << 14;
// 512 bytes of scales (32 rows of 16 bytes, eight rows 128 bytes apart) into four columns of tensor memory, the same in
// every quarter of the lanes
template <int CTAS>
__device__ __forceinline__ void scales_to_tmem(unsigned tmem, unsigned lo) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(from_words(lo, SCALE_HI)) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(from_words(lo, SCALE_HI)) : "memory");
}
#define MX4_MMA(GROUP, KIND_VEC)                                                                                                   \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                                  \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND_VEC " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"                          \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory")
template <int KIND, int CTAS>
__device__ __forceinline__ void umma_scaled(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa,
                                            unsigned sb, unsigned accumulate) {
    if constexpr (KIND != CODES && CTAS == 1) MX4_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (KIND != CODES) MX4_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (CTAS == 1) MX4_MMA("1", "mxf4.block_scale.scale_vec::2X");
    else MX4_MMA("2", "mxf4.block_scale.scale_vec::2X");
}
#undef MX4_MMA

// the plan of a stage's shared and tensor memory
template <int KIND, int BN> struct Plan {
    static constexpr int TOKENS = BN / KIND, PART = TOKENS + 4;          // of a tile; of a row of W's part of the sums, with room against bank conflicts
    static constexpr int B_BYTES = BN * 128;
    static constexpr int K_TILES = KIND != CODES ? 1 : 2;                // 128-column tiles of scales a stage
    static constexpr int B_GROUPS = (BN + 127) / 128;                    // 128-row tiles of scales
    static constexpr int SA_BYTES = 512 * K_TILES, SB_BYTES = 512 * K_TILES * B_GROUPS;
    static constexpr int SCALE_COLS = 4 * K_TILES * (1 + B_GROUPS);      // of tensor memory a stage
    static_assert(KIND != PIECES_F32 || BN % 80 == 0, "read back sixteen tokens at a time");
    static constexpr int tmem_cols(int stages) {
        int c = 32;
        while (c < BN + stages * SCALE_COLS) c *= 2;
        return c;
    }
};

__device__ __forceinline__ void store(const Params& p, int t, int f, float v) {
    if (p.y_is_f32) reinterpret_cast<float*>(p.y)[(long)t * p.ldy + f] = v;
    else reinterpret_cast<__nv_bfloat16*>(p.y)[(long)t * p.ldy + f] = __float2bfloat16_rn(v);
}

// One stage's products, issued by one thread: scales into the stage's columns of tensor memory (`scales`), then four products
// of 32 bytes of each row: 32 numbers spread to bytes, or 64 packed ones.  a, b, sa, sb: where the stage's tiles start, in units of
// 16 bytes; shift: columns of scales in front of x's.
template <int KIND, int BN, int CTAS>
__device__ __forceinline__ void multiply_stage(unsigned tmem, unsigned scales, unsigned a, unsigned b, unsigned sa_tile, unsigned sb_tile,
                                               bool accumulate, unsigned shift = 0) {
    using P = Plan<KIND, BN>;
    constexpr unsigned FORMATS = KIND != CODES ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);   // e2m1 and e4m3, e2m1 twice
    constexpr unsigned IDESC = FORMATS | ((unsigned)(BN >> 3) << 17) | (1u << 23) | ((unsigned)(CTAS * BM >> 4) << 24);
    const unsigned sa = scales, sb = sa + 4 * P::K_TILES;
#pragma unroll
    for (int j = 0; j < P::K_TILES; ++j) {
        scales_to_tmem<CTAS>(sa + 4 * j, sa_tile + 32 * j);
#pragma unroll
        for (int g = 0; g < P::B_GROUPS; ++g)     // the column tiles one after the other, the row tiles of each side by side
            scales_to_tmem<CTAS>(sb + 4 * (j * P::B_GROUPS + g), sb_tile + g * (P::SA_BYTES / 16) + 32 * j);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned tile = KIND != CODES ? 0 : k >> 1, id = KIND != CODES ? k : (k & 1) * 2;
        umma_scaled<KIND, CTAS>(tmem, from_words(TILE_LO + a + 2 * k, TILE_HI), from_words(TILE_LO + b + 2 * k, TILE_HI),
                          IDESC | (id << 4) | (id << 29), sa + 4 * tile, sb + 4 * P::B_GROUPS * tile + shift, accumulate || k != 0);
    }
}

__device__ __forceinline__ unsigned f16_pair(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
// two numbers (f16) to their first pieces and 32 times what they leave of them to the second ones
__device__ __forceinline__ void two_pieces(unsigned v, unsigned short& first, unsigned short& second) {
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(first) : "r"(v));
    const unsigned back = few::values8x2(first);
    const __half2 k32 = __float2half2_rn(32.0f);
    const __half2 left = __hmul2(k32, __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&back)));
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(second) : "r"(*reinterpret_cast<const unsigned*>(&left)));
}

template <int COLUMNS>
__device__ __forceinline__ void tmem_columns(unsigned from, unsigned (&r)[COLUMNS]) {
#pragma unroll
    for (int c = 0; c < COLUMNS / 16; ++c)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(r[16 * c]), "=r"(r[16 * c + 1]), "=r"(r[16 * c + 2]), "=r"(r[16 * c + 3]), "=r"(r[16 * c + 4]), "=r"(r[16 * c + 5]),
                       "=r"(r[16 * c + 6]), "=r"(r[16 * c + 7]), "=r"(r[16 * c + 8]), "=r"(r[16 * c + 9]), "=r"(r[16 * c + 10]), "=r"(r[16 * c + 11]),
                       "=r"(r[16 * c + 12]), "=r"(r[16 * c + 13]), "=r"(r[16 * c + 14]), "=r"(r[16 * c + 15])
                     : "r"(from + 16 * c));
    tmem_ld_wait();
}

constexpr int STORE_BYTES = 4096;      // a warp's piece of shared memory for results on their way out
// A warp stores `count` tokens' results of up to 32 rows of W from f0 on, those below `end`, a lane a row: through shared memory, so that
// a token's results go out in pieces of 16 bytes where y allows it (4,096 x 4,096 and 48 rows: 13.0 us, number by
// number 15.5).
template <typename T, int COUNT>
__device__ __forceinline__ void store_rows(const Params& p, unsigned char* mine, const float (&v)[COUNT], int t0, int count, int f0, int end, int lane) {
    T* rows = reinterpret_cast<T*>(mine);
    static_assert(COUNT * 32 * sizeof(T) <= STORE_BYTES, "a warp's piece");
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        if constexpr (sizeof(T) == 4) rows[32 * j + lane] = v[j];
        else rows[32 * j + lane] = __float2bfloat16_rn(v[j]);
    }
    __syncwarp();
    constexpr int LANES = 2 * sizeof(T), PER = 32 / LANES, PIECE = 16 / (int)sizeof(T);      // lanes that a token's results take, tokens at a time
    T* y = reinterpret_cast<T*>(p.y) + (long)t0 * p.ldy + f0;
    if (p.y_wide && (end - f0 >= 32 || end % PIECE == 0)) {
        const int r = lane / LANES, c = lane % LANES * PIECE;
#pragma unroll
        for (int j = 0; j < COUNT; j += PER)
            if (j + r < count && f0 + c < end) *reinterpret_cast<uint4*>(y + (long)(j + r) * p.ldy + c) = *reinterpret_cast<const uint4*>(rows + 32 * (j + r) + c);
    } else if (f0 + lane < end) {
        for (int j = 0; j < count; ++j) y[(long)j * p.ldy + lane] = rows[32 * j + lane];
    }
    __syncwarp();
}

// ---- up to 64 rows: what counts is that every SM streams its share of the weights -----------------------------------------------
// A tile may cover fewer rows of W than the product's 128 (a multiple of eight; what the tensor core reads beyond them belongs
// to other tiles and its results are not stored), so that the tiles can be as many as the SMs, or twice as many.  Its scales are then
// not a 512-byte tile of the matrix's: helper warps put them together, a warp every fourth stage's, and, where the kernel brings
// x's numbers to pieces itself, two warps every fourth stage's pieces.
__device__ __forceinline__ void copy4(unsigned dst, const void* src, bool in) {        // four bytes, or zeros
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// the thread's arrival at a barrier when its copies so far are there (counted in the barrier's arrivals)
__device__ __forceinline__ void arrive_with_copies(unsigned bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

struct Shape {
    int tile_rows, stages, splits, tmem_cols;
    int x_rows;      // columns of the products that are brought: one tile of tokens alone needs no more than x has (the rest are not stored)
};

// (INSIDE) A thread takes eight numbers of a row of x, four threads a block of 32, a warp two rows; what it needs of its next stage is on
// its way.  The numbers go through f16, which holds a
// bfloat16 number's eight bits from 256 down to 2^-17 and below that what the second piece may still need.
template <int KIND, int BN, bool INSIDE>
__device__ __forceinline__ bool fill_stages(const Params& p, const Shape& sh, int row0, unsigned char* b_tiles, unsigned char* sa_tiles,
                                            unsigned char* sb_tiles, int kb0, int nkb, unsigned full0, unsigned empty0) {
    using P = Plan<KIND, BN>;
    const int which = (int)(threadIdx.x - THREADS) >> 5, half = which >> 2;
    const int lane = threadIdx.x & 31, g = lane & 15, t = 2 * half + (lane >> 4), rows = (p.n_out + 127) / 128 * 128 - row0;      // of scales there are
    const unsigned* scales = reinterpret_cast<const unsigned*>(p.w_scales);
    // a stage's scales are on their way with its weights (the weights' scales come from as far as the weights do)
    auto fetch_scales = [&](int i, int s) {
#pragma unroll
        for (int j = 0; j < P::K_TILES; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = 32 * c + lane;
                const bool in = r < sh.tile_rows && r < rows;
                copy4(smem_u32(sa_tiles + s * P::SA_BYTES + 512 * j + 16 * lane + 4 * c),
                      scales + (in ? few::scale_word(row0 + r, (kb0 + i) * P::K_TILES + j, p.scale_tiles) : 0), in);
            }
        arrive_with_copies(full0 + 8 * s);
    };
    // No more helpers than stages: a warp that has filled stage i knows the products of stage i - stages done; its next stage's
    // place was last but one used by stage i + helpers - 2 stages, and only if that one is done too does the parity of the place's
    // barrier say which use it speaks of.
    const int helpers = sh.stages < 4 ? sh.stages : 4;
    int i = which & 3;
    if (i >= helpers) return true;
    for (int a = i; half == 0 && a < nkb && a < sh.stages; a += helpers) fetch_scales(a, a);      // before the kernel ahead is done
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint4 raw;
    const __nv_bfloat16* x = ib_after_wait(reinterpret_cast<const __nv_bfloat16*>(p.x) + (long)t * p.ldx + 8 * g);
    auto fetch_x = [&](int i) {
        const int c = (kb0 + i) * 128, n = p.k - c - 8 * g;
        raw = make_uint4(0, 0, 0, 0);
        if (t >= p.n_tok || i >= nkb) return;
        if (p.wide && n >= 8) {
            raw = *reinterpret_cast<const uint4*>(x + c);
        } else {
            unsigned short* to = reinterpret_cast<unsigned short*>(&raw);
#pragma unroll
            for (int e = 0; e < 8; ++e) if (e < n) to[e] = *reinterpret_cast<const unsigned short*>(x + c + e);
        }
    };
    if constexpr (INSIDE) fetch_x(i);
    int s = i;
    unsigned phase = 1;                  // of the place's barrier at this stage's turn
    for (; i < nkb; i += helpers, s += helpers) {
        if (s >= sh.stages) { s -= sh.stages; phase ^= 1; }
        if (i >= sh.stages && !mbar_wait(empty0 + 8 * s, phase, 4)) return false;
        if (half == 0 && i >= sh.stages) fetch_scales(i, s);
        if constexpr (INSIDE) {
            if (2 * half < p.n_tok) {      // (else columns of no token: whatever the stage holds)
                const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
                unsigned m = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & 0x7FFF7FFFu);
                m = max(m & 0xFFFFu, m >> 16);
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const unsigned byte = few::pieces_byte<PIECES_BF16>(m << 16);
                const float by = byte == 255u ? 0.0f : few::scale_reciprocal(byte);
                unsigned short h[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    two_pieces(byte == 255u ? 0u : f16_pair(__uint_as_float(w[e] << 16) * by, __uint_as_float(w[e] & 0xFFFF0000u) * by), h[e], l[e]);
                const int r = 2 * t;
                unsigned char* to = b_tiles + s * P::B_BYTES + (g & 1) * 8;
                *reinterpret_cast<uint2*>(to + r * 128 + ((g >> 1) ^ (r & 7)) * 16) = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
                *reinterpret_cast<uint2*>(to + (r + 1) * 128 + ((g >> 1) ^ ((r + 1) & 7)) * 16) = make_uint2(l[0] | (unsigned)l[1] << 16, l[2] | (unsigned)l[3] << 16);
                if ((lane & 3) == 0) {
                    unsigned char* sc = sb_tiles + s * P::SB_BYTES + r * 16 + (g >> 2);
                    sc[0] = (unsigned char)byte;
                    sc[16] = (unsigned char)(byte == 255u ? 255u : byte - 5u);
                }
            }
            fetch_x(i + helpers);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the tensor core reads them behind the barrier
            __syncwarp();
            if (lane == 0) mbar_arrive(full0 + 8 * s);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return true;
}

// INSIDE: the kernel brings x's rows to pieces itself
template <int KIND, int BN, bool INSIDE>
__global__ void __launch_bounds__(THREADS + (INSIDE ? 256 : 128)) few_rows_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                 const __grid_constant__ CUtensorMap map_x, const Params p, const Shape sh) {
    using P = Plan<KIND, BN>;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
    const int stages = sh.stages, splits = sh.splits, a_bytes = sh.tile_rows * 128;
    unsigned char* b_tiles = smem;
    unsigned char* a_tiles = b_tiles + stages * P::B_BYTES;
    unsigned char* sa_tiles = a_tiles + stages * a_bytes;
    unsigned char* sb_tiles = sa_tiles + stages * P::SA_BYTES;
    float* recv = reinterpret_cast<float*>(sb_tiles + stages * P::SB_BYTES);     // [rank of the sender][rows owned][TOKENS, and four of room]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(reinterpret_cast<unsigned char*>(recv) + (splits > 1 ? P::PART * sh.tile_rows * 4 : 0));
    const unsigned full0 = smem_u32(bars), empty0 = smem_u32(bars + stages), accum = smem_u32(bars + 2 * stages);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 2 * stages + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * sh.tile_rows, tile_t = blockIdx.y;
    const int kb0 = (int)((long)blockIdx.z * p.num_kb / splits), nkb = (int)((long)(blockIdx.z + 1) * p.num_kb / splits) - kb0;   // >= 1

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(full0 + 8 * s, INSIDE ? 35 : 33); mbar_init(empty0 + 8 * s, 1); }
        mbar_init(accum, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(sh.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    // (not before: a CTA of the next kernel that came first could hold columns that this one waits for, and wait for its end)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    fence_after();
    const unsigned tmem = *tmem_slot;
    bool ok = true;
    if (p.wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (splits > 1) cluster_arrive();       // "this CTA runs": looked at before the first store to it

    if (warp == 0) {
        const bool leader = elected();
        const unsigned long long pol = policy_evict_first();
        const unsigned w_tx = KIND == CODES ? a_bytes : a_bytes / 2;     // what a tile of weights counts on its barrier
        auto load_w = [&](int i, int s) {
            if (!leader) return;
            mbar_expect_tx(full0 + 8 * s, w_tx + (INSIDE ? 0 : sh.x_rows * 128 + P::SB_BYTES));
            tma_load_2d_hint(smem_u32(a_tiles) + s * a_bytes, &map_w, (kb0 + i) * 128, row0, full0 + 8 * s, pol);
        };
        auto load_x = [&](int i, int s) {
            if (INSIDE || !leader) return;
            tma_load_2d(smem_u32(b_tiles) + s * P::B_BYTES, &map_x, (kb0 + i) * 128, tile_t * BN, full0 + 8 * s);
#pragma unroll
            for (int g = 0; g < P::B_GROUPS; ++g)
                bulk_load(smem_u32(sb_tiles) + s * P::SB_BYTES + g * P::SA_BYTES,
                          p.x_scales + ((long)(tile_t * P::B_GROUPS + g) * p.scale_tiles + (long)(kb0 + i) * P::K_TILES) * 512,
                          P::SA_BYTES, full0 + 8 * s);
        };
        const int head = nkb < stages ? nkb : stages;    // the first weights are on their way before the kernel ahead is done
        for (int i = 0; i < head; ++i) load_w(i, i);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int i = 0; i < head; ++i) load_x(i, i);
        unsigned phase = 0;
        for (int i = head, s = 0; i < nkb; ++i) {
            if (!mbar_wait(empty0 + 8 * s, phase, 1)) { ok = false; break; }
            load_w(i, s);
            load_x(i, s);
            if (++s == stages) { s = 0; phase ^= 1; }
        }
    } else if (warp == 1) {
        const bool leader = elected();
        const unsigned a0 = smem_u32(a_tiles) >> 4, b0 = smem_u32(b_tiles) >> 4, sa0 = smem_u32(sa_tiles) >> 4, sb0 = smem_u32(sb_tiles) >> 4;
        unsigned phase = 0;
        for (int i = 0, s = 0; i < nkb; ++i) {
            if (!mbar_wait(full0 + 8 * s, phase, 2)) { ok = false; break; }
            fence_after();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the scales came by plain copies
            if (leader) {
                multiply_stage<KIND, BN, 1>(tmem, tmem + BN + s * P::SCALE_COLS, a0 + s * (a_bytes >> 4), b0 + s * (P::B_BYTES / 16),
                                         sa0 + s * (P::SA_BYTES / 16), sb0 + s * (P::SB_BYTES / 16), i != 0);
                umma_commit(empty0 + 8 * s);
            }
            if (++s == stages) { s = 0; phase ^= 1; }
        }
        if (leader) umma_commit(accum);
    } else if (warp >= 6) {
        ok = fill_stages<KIND, BN, INSIDE>(p, sh, row0, b_tiles, sa_tiles, sb_tiles, kb0, nkb, full0, empty0);
    }

    const int q = warp & 3, row = q * 32 + lane;
    const unsigned rank = blockIdx.z;
    const int owned = sh.tile_rows / splits;           // rows of the tile that a CTA of the cluster adds up and stores
    const int t0 = tile_t * P::TOKENS, tokens = p.n_tok - t0 < P::TOKENS ? p.n_tok - t0 : P::TOKENS;
    const int rows = p.n_out - row0 < sh.tile_rows ? p.n_out - row0 : sh.tile_rows;
    if (splits > 1) cluster_wait();
    if (warp >= 2 && warp < 6) {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // y may still be read by the kernel ahead
        ok = mbar_wait(accum, 0, 3);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
        if (ok && g_error == 0 && q * 32 < sh.tile_rows) {
            // accumulator columns at a time, their tokens; the stages' shared memory is free (one stage has what a warp's tokens take for every 32
            // rows begun: 4 KB where B's tile does, 2 KB at most with 16 columns)
            constexpr int COLS = KIND == PIECES_F32 ? 80 : BN < 32 ? BN : 32, STEP = COLS / KIND;
            unsigned char* mine = smem + q * STORE_BYTES;
            const unsigned there = splits > 1 ? at_rank(smem_u32(recv + ((size_t)rank * owned + row % owned) * P::PART), (unsigned)(row / owned % splits)) : 0;
#pragma unroll 1
            for (int c = 0; c * STEP < tokens; ++c) {
                unsigned r[COLS];
                __syncwarp();      // rows beyond the tile's skip the stores
                tmem_columns<COLS>(tmem + ((unsigned)(q * 32) << 16) + COLS * c, r);
                float v[STEP];
#pragma unroll
                for (int j = 0; j < STEP; ++j) {
                    v[j] = 0.0f;
#pragma unroll
                    for (int i = KIND - 1; i >= 0; --i) v[j] += __uint_as_float(r[KIND * j + i]);
                }
                if (splits > 1) {
#pragma unroll
                    for (int j = 0; j < STEP; j += 4)
                        if (row < sh.tile_rows && c * STEP + j < tokens) st_remote_f32x4(there + 4 * (c * STEP + j), v[j], v[j + 1], v[j + 2], v[j + 3]);
                } else {
                    const int count = tokens - c * STEP < STEP ? tokens - c * STEP : STEP;
                    if (p.y_is_f32) store_rows<float, STEP>(p, mine, v, t0 + c * STEP, count, row0 + q * 32, row0 + rows, lane);
                    else store_rows<__nv_bfloat16, STEP>(p, mine, v, t0 + c * STEP, count, row0 + q * 32, row0 + rows, lane);
                }
            }
        }
    }
    if (splits > 1) {
        cluster_arrive();
        cluster_wait();                      // every part of the rows that this CTA owns is in its shared memory
        if (warp >= 2 && warp < 6 && g_error == 0) {
            for (int i = (int)threadIdx.x - 64; i < (tokens + 3) / 4 * owned; i += 128) {
                const int t = i / owned * 4, r = i % owned, f = (int)rank * owned + r;
                if (f >= rows) continue;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int part = 0; part < splits; ++part) {
                    const float4 v = *reinterpret_cast<const float4*>(recv + ((size_t)part * owned + r) * P::PART + t);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                store(p, t0 + t, row0 + f, sum.x);
                if (t + 1 < tokens) store(p, t0 + t + 1, row0 + f, sum.y);
                if (t + 2 < tokens) store(p, t0 + t + 2, row0 + f, sum.z);
                if (t + 3 < tokens) store(p, t0 + t + 3, row0 + f, sum.w);
            }
        }
    }
    // after a wait that ran out the copies in flight are given time to land before the shared memory is given back
    if (!ok) for (const unsigned long long t = global_ns(); global_ns() - t < 20000000ull;) {}
    fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(sh.tmem_cols));
}

// ---- more rows ------------------------------------------------------------------------------------------------------------------
// A pair of CTAs (a cluster) multiplies 256 rows of W with one tile of tokens: each loads its own 128 rows and half of the tokens, the
// first one issues products that read the shared memories of both and leave each CTA its own rows' results. The halves are what
// counts: an SM's shared memory moves 128 bytes a cycle, and a stage of 128 x 192 alone has it take in and read out 64 KB (4-bit weights
// and pieces) or 80 KB (4-bit rows), 512 and 640 cycles where the products take 384 (measured: 500 and 650); here it is 40 and 56 KB.
// The pairs stay and take tile after tile; two accumulators take turns, so that four warps read one back and store it while the
// other is being filled.  A stage then takes 395 cycles (pieces) and 410 .. 490 (4-bit rows, 28 KB a CTA from L2), and what bounds it is the clock
// at which the tensor cores run under load, 1.3 to 1.6 GHz: 2,048 x 12,288 x 4,096 (bfloat16 rows) 130 us behind the 29 that bring x to
// pieces, 3.2 PFLOP/s of 8-bit products (CTAs by themselves, one tile each: 170); 4-bit rows 2,048 x 4,096 x 24,576 72 to 81 us, 5.1 to 5.7
// PFLOP/s (200).  Four CTAs that share x's tiles have room on 132 SMs and gain nothing.
constexpr int PAIR = 2;
template <int KIND, int BN, int STAGES> struct Many {
    using P = Plan<KIND, BN>;
    static constexpr int B_BYTES = P::B_BYTES / PAIR;
    static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES + P::SA_BYTES + P::SB_BYTES) + 4 * STORE_BYTES + 16 * STAGES + 64 + 1024;
    static_assert(2 * BN + STAGES * P::SCALE_COLS <= 512 && SMEM <= 227 * 1024 && SMEM > 114 * 1024, "memories of an SM");
    static_assert(BN % 32 == 0 && BN / PAIR % 8 == 0, "halves of a tile are whole groups of eight rows");
};
// one arrival at the barrier of either CTA when the products so far are done
__device__ __forceinline__ void umma_commit_pair(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((unsigned short)3) : "memory");
}
// (relaxed: what it tells of is in registers; a release would wait for the results on their way to y)
__device__ __forceinline__ void arrive_there(unsigned bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// into this CTA's shared memory, counted on a barrier of either CTA
__device__ __forceinline__ void tma_load_2d_pair(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

template <int KIND, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS + 32) gemm_kernel(const __grid_constant__ CUtensorMap map_w,
                                                            const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_sw,
                                                            const __grid_constant__ CUtensorMap map_sx, const Params p) {
    using P = Plan<KIND, BN>;
    using M = Many<KIND, BN, STAGES>;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
    unsigned char* a_tiles = smem;
    unsigned char* b_tiles = a_tiles + STAGES * A_BYTES;
    unsigned char* sa_tiles = b_tiles + STAGES * M::B_BYTES;
    unsigned char* sb_tiles = sa_tiles + STAGES * P::SA_BYTES;
    unsigned char* stores = sb_tiles + STAGES * P::SB_BYTES;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(stores + 4 * STORE_BYTES);
    // full (the first CTA's): a stage has landed in both; empty: the products are done with it; filled: an accumulator holds a tile; drained
    // (the first CTA's): both have read theirs
    const unsigned full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), filled0 = smem_u32(bars + 2 * STAGES), drained0 = filled0 + 16;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 2 * STAGES + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nkb = p.num_kb;
    const int rank = blockIdx.x & 1, pairs_f = (p.n_out + PAIR * BM - 1) / (PAIR * BM), tiles = pairs_f * ((p.n_tok + P::TOKENS - 1) / P::TOKENS);
    const int first = blockIdx.x / PAIR, step = gridDim.x / PAIR, stages = (tiles - first + step - 1) / step * nkb;      // of this pair
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 2); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(filled0 + 8 * b, 1); mbar_init(drained0 + 8 * b, 4 * PAIR); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    // (not before: a CTA of the next kernel that came first could hold columns that this one waits for, and wait for its end)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cluster_arrive();      // nothing is sent to the other CTA before its barriers stand
    cluster_wait();
    fence_after();
    const unsigned tmem = *tmem_slot;
    bool ok = true;
    if (p.wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");
    // Copies are issued by two threads a CTA, one for the operands and one for their scales; those of the first CTA announce what both bring.
    if (warp == 0 || warp == 6) {
        const bool leader = elected(), operands = warp == 0;
        constexpr unsigned W_TX = KIND != CODES ? A_BYTES / 2 : A_BYTES;     // what a tile of weights counts on its barrier
        const unsigned full = at_rank(full0, 0);
        int tile = first, tile_f = 0, row_x = 0, group = 0;
        auto enter = [&]() {      // (what lies behind the last rows reads as zeros)
            const int tile_t = tile / pairs_f;
            tile_f = tile % pairs_f * PAIR + rank;
            row_x = tile_t * BN + rank * (BN / PAIR);
            group = KIND == CODES ? tile_t * BN / 128 : tile_t * P::B_GROUPS;
        };
        auto load_w = [&](int i, int s) {
            if (!leader) return;
            if (operands) {
                if (rank == 0) mbar_expect_tx(full0 + 8 * s, PAIR * (W_TX + M::B_BYTES));
                tma_load_2d_pair(smem_u32(a_tiles) + s * A_BYTES, &map_w, i * 128, tile_f * BM, full + 8 * s);
            } else {
                if (rank == 0) mbar_expect_tx(full0 + 8 * s, PAIR * (P::SA_BYTES + P::SB_BYTES));
                tma_load_3d_pair(smem_u32(sa_tiles) + s * P::SA_BYTES, &map_sw, 0, i * P::K_TILES, tile_f, full + 8 * s);
            }
        };
        auto load_x = [&](int i, int s) {
            if (!leader) return;
            if (operands) tma_load_2d_pair(smem_u32(b_tiles) + s * M::B_BYTES, &map_x, i * 128, row_x, full + 8 * s);
            else tma_load_3d_pair(smem_u32(sb_tiles) + s * P::SB_BYTES, &map_sx, 0, i * P::K_TILES, group, full + 8 * s);      // (every CTA's rows meet all tokens)
        };
        const int head = nkb < STAGES ? nkb : STAGES;    // the first weights are on their way before the kernel ahead is done
        enter();
        for (int i = 0; i < head; ++i) load_w(i, i);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int i = 0;
        unsigned phase = 1;
        for (int it = 0; it < stages && ok; it += STAGES, phase ^= 1) {
#pragma unroll
            for (int s = 0; s < STAGES; ++s) {
                if (it + s >= stages) break;
                if (it + s >= head) {
                    if (!mbar_wait(empty0 + 8 * s, phase, 1)) { ok = false; break; }
                    load_w(i, s);
                }
                load_x(i, s);
                if (++i == nkb) { i = 0; tile += step; enter(); }
            }
        }
        // the last arrivals have come: none is on its way to a CTA that has ended
        for (int s = 0; ok && s < STAGES; ++s) {
            const int uses = (stages - s + STAGES - 1) / STAGES;
            ok = uses == 0 || mbar_wait(empty0 + 8 * s, (uses - 1) & 1, 1);
        }
    } else if (warp == 1 && rank == 0) {
        const bool leader = elected();
        const unsigned a0 = smem_u32(a_tiles) >> 4, b0 = smem_u32(b_tiles) >> 4, sa0 = smem_u32(sa_tiles) >> 4, sb0 = smem_u32(sb_tiles) >> 4;
        // a tile of 4-bit rows may start amid a tile of 128 rows of scales, 32 of them a column
        auto shift_of = [&](int tile) { return KIND == CODES ? (unsigned)(tile / pairs_f * BN / 32 & 3) : 0u; };
        int i = 0, tile = first;
        unsigned phase = 0, turn = 0, shift = shift_of(tile);
        bool landed = mbar_try_wait(full0, 0);      // the next stage's answer is on its way while a stage is issued
        for (int it = 0; it < stages && ok; it += STAGES, phase ^= 1) {
#pragma unroll
            for (int s = 0; s < STAGES; ++s) {
                if (it + s >= stages) break;
                const unsigned buffer = turn & 1;
                if (i == 0 && !mbar_wait(drained0 + 8 * buffer, (turn >> 1 & 1) ^ 1, 4)) { ok = false; break; }
                if (!landed && !mbar_wait(full0 + 8 * s, phase, 2)) { ok = false; break; }
                landed = mbar_test_wait(full0 + 8 * ((s + 1) % STAGES), s + 1 == STAGES ? phase ^ 1 : phase);
                fence_after();
                if (leader) {
                    multiply_stage<KIND, BN, PAIR>(tmem + buffer * BN, tmem + 2 * BN + s * P::SCALE_COLS, a0 + s * (A_BYTES / 16), b0 + s * (M::B_BYTES / 16),
                                             sa0 + s * (P::SA_BYTES / 16), sb0 + s * (P::SB_BYTES / 16), i != 0, shift);
                    umma_commit_pair(empty0 + 8 * s);
                    if (i == nkb - 1) umma_commit_pair(filled0 + 8 * buffer);
                }
                if (++i == nkb) { i = 0; tile += step; ++turn; shift = shift_of(tile); }
            }
        }
    } else if (warp != 1) {
        const int q = warp & 3;
        unsigned char* mine = stores + q * STORE_BYTES;
        asm volatile("griddepcontrol.wait;" ::: "memory");   // y may still be read by the kernel ahead
        int turn = 0;
        for (int tile = first; tile < tiles; tile += step, ++turn) {
            const unsigned buffer = turn & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(filled0 + 8 * buffer, turn >> 1 & 1, 3)) && *(volatile int*)&g_error == 0;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const int f0 = (tile % pairs_f * PAIR + rank) * BM + q * 32, t0 = tile / pairs_f * P::TOKENS;
            const int tokens = p.n_tok - t0 < P::TOKENS ? p.n_tok - t0 : P::TOKENS;
            constexpr int STEP = KIND == PIECES_F32 ? 16 : 32 / KIND, COLUMNS = STEP * KIND;      // tokens and columns at a time
#pragma unroll 1
            for (int c = 0; c * STEP < tokens; ++c) {
                unsigned r[COLUMNS];
                const unsigned from = tmem + buffer * BN + ((unsigned)(q * 32) << 16) + COLUMNS * c;
                tmem_columns<COLUMNS>(from, r);
                float v[STEP];
#pragma unroll
                for (int j = 0; j < STEP; ++j) {
                    v[j] = 0.0f;
#pragma unroll
                    for (int i = KIND - 1; i >= 0; --i) v[j] += __uint_as_float(r[KIND * j + i]);
                }
                if ((c + 1) * STEP >= tokens) {      // all is in registers
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_there(at_rank(drained0 + 8 * buffer, 0));
                }
                const int count = tokens - c * STEP < STEP ? tokens - c * STEP : STEP;
                if (f0 >= p.n_out) continue;
                if (p.y_is_f32) store_rows<float, STEP>(p, mine, v, t0 + c * STEP, count, f0, p.n_out, lane);
                else store_rows<__nv_bfloat16, STEP>(p, mine, v, t0 + c * STEP, count, f0, p.n_out, lane);
            }
        }
    }
    // after a wait that ran out the copies in flight are given time to land before the shared memory is given back
    if (!ok) for (const unsigned long long t = global_ns(); global_ns() - t < 20000000ull;) {}
    fence_before();
    __syncthreads();
    cluster_arrive();      // the other CTA may still be told that this one is done with a stage, or send to it
    cluster_wait();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Where the scales of a row's first piece stand: the pieces of a tile of tokens have tiles of 128 rows of scales of their own.
template <int PARTS> __host__ __device__ __forceinline__ int pieces_scale_row(int row, int tokens) {
    return row / tokens * ((tokens * PARTS + 127) / 128 * 128) + row % tokens * PARTS;
}
// Rows as pieces: row PARTS * t + i of `pieces` [PARTS * n, kp] holds piece i of row t, kp = width rounded up to 128.  A
// warp takes 256 columns of one or two rows: a lane eight numbers, four lanes a block of 32, sixteen a word of four scales.  Memory
// bounds it where the conversions leave it time: 2,048 x 12,288 bfloat16 numbers, 101 MB, 29 us with two rows, 33 with one; where
// warps of one row do not fill the SMs, one is faster (512 x 4,096 4.6 and 5.3 us, 128 x 4,096 3.0 and 3.4).
constexpr int PIECES_WARPS = 8;
template <typename T, int PARTS, int PIECES_ROWS>
__global__ void __launch_bounds__(32 * PIECES_WARPS) pieces_kernel(const T* __restrict__ x, long ldx, int rows, int width, int tokens,
                                                     uint2* __restrict__ pieces, unsigned* __restrict__ scales) {
    ib_grid_dependency_sync();
    x = ib_after_wait(x);
    const few::Strip at(width, PIECES_ROWS);
    const int row0 = at.row0, g = at.g, per_row = (width + 127) / 128 * 16, tiles = few::scale_tiles(width), lane = threadIdx.x & 31;
    few::Eight<T> raw[PIECES_ROWS];
#pragma unroll
    for (int r = 0; r < PIECES_ROWS; ++r) {
        const bool in = row0 + r < rows;
        raw[r].load(x + (long)(in ? row0 + r : 0) * ldx + at.column, in ? width - at.column : 0);
    }
#pragma unroll
    for (int r = 0; r < PIECES_ROWS; ++r) {
        const unsigned byte = few::pieces_byte<PARTS>(few::block_largest(raw[r].largest()));
        const float by = byte == 255u ? 0.0f : few::scale_reciprocal(byte);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = byte == 255u ? 0.0f : raw[r][j] * by;
        uint2 c[PARTS];
        if constexpr (PARTS == PIECES_BF16) {
            unsigned short h[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) two_pieces(f16_pair(v[2 * j], v[2 * j + 1]), h[j], l[j]);
            c[0] = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
            c[1] = make_uint2(l[0] | (unsigned)l[1] << 16, l[2] | (unsigned)l[3] << 16);
        } else {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) c[part] = few::take_piece(v);
        }
        unsigned word = byte << (8 * (lane >> 2 & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (row0 + r >= rows || g >= per_row) continue;
        const int first = pieces_scale_row<PARTS>(row0 + r, tokens);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            pieces[((long)(row0 + r) * PARTS + part) * per_row + g] = c[part];
            // every further piece's byte is five less; 255 stays (no byte is below five times the pieces in front of its own)
            if ((lane & 15) == 0) scales[few::scale_word(first + part, g >> 4, tiles)] = __vsub4(word, __vcmpne4(word, 0xFFFFFFFFu) & (0x01010101u * (5 * part)));
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long inner, long rows, long row_bytes, int box_inner, int box_rows) {
    EncodeTiled fn = encode_fn();
    if (fn == nullptr) return IB_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? IB_OK : IB_ERR_UNSUPPORTED;
}

// the tensor maps of both operands: weights in boxes of box_w rows, x (not where it is brought to pieces inside) of box_x
template <int KIND>
static int make_maps(CUtensorMap* map_w, CUtensorMap* map_x, const void* w, const void* x, int n, int m, int k, int box_w, int box_x, Params& p) {
    const long kp = (long)(k + 127) / 128 * 128;
    p.scale_tiles = few::scale_tiles(k);
    p.num_kb = (int)(KIND != CODES ? kp / 128 : (kp + 255) / 256);
    int r = KIND != CODES ? make_map(map_w, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, w, kp, m, kp / 2, 128, box_w)
                          : make_map(map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, kp / 2, m, kp / 2, 128, box_w);
    if (r || x == nullptr) { *map_x = *map_w; return r; }
    return KIND != CODES ? make_map(map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, kp, (long)KIND * n, kp, 128, box_x)
                         : make_map(map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, kp / 2, n, kp / 2, 128, box_x);
}

// tiles of 512 bytes of scales, `tiles` for each of `groups` tiles of 128 rows, in boxes of box_tiles by box_groups
static int make_scale_map(CUtensorMap* map, const void* base, int tiles, int groups, int box_tiles, int box_groups) {
    EncodeTiled fn = encode_fn();
    if (fn == nullptr) return IB_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {128, (cuuint64_t)tiles, (cuuint64_t)groups}, strides[2] = {512, (cuuint64_t)tiles * 512};
    cuuint32_t box[3] = {128, (cuuint32_t)box_tiles, (cuuint32_t)box_groups}, step[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? IB_OK : IB_ERR_UNSUPPORTED;
}

constexpr int SMS = 148, FEW_SMEM = 100 * 1024, ALONE_SMEM = 200 * 1024;      // of a CTA of the kernel for few rows: two share an SM, or one has it

// How the weights of a product of few rows are cut: into tiles of at most 128 rows, or K into parts.  A CTA takes 350 cycles a stage
// (the issue of its copies and products), what its bytes take at 42 a cycle, or the tensor core's time, after a start of 2,750; two
// share an SM; its results cost 80 cycles a row of x, and parts their meeting, which grows with the rows of x too.  The numbers are
// fitted to 4,700 products of 20 kinds (six matrices, 1 to 64 rows, every height and cut): what the rule takes is 3 % slower than the
// best on average (lowered tiles in parts as well: 3.5 %).  Us of a product in a row of products, tiles x parts: 4,096 x 4,096, one row 128 x 1 9.4, 64 x 2 7.7, 128 x 4 6.2,
// 128 x 8 6.7; 64 rows 128 x 1 14.9, 64 x 2 12.0, 128 x 4 10.2.  4,096 x 24,576, one row: 88 x 1 12.5, 128 x 1 12.8; 64 rows 19.0, 22.9.  (More than four
// rows: as in captured steps; a call that waits for the rows' way to pieces takes about 1 us more, with every shape.)
template <int KIND, int BN>
static Shape shape_for(int n, int m, int num_kb, int tiles_t, int tile_rows, int splits) {
    using P = Plan<KIND, BN>;
    auto lowered = [](long rows) { return rows > 128 ? 128 : (int)(rows + 7) / 8 * 8; };
    // (as many as a whole tile: float32, 4,096 x 24,576, six rows 28 us, seven 18; like this 16)
    Shape s = {tile_rows > 0 ? tile_rows : 128, 1, splits > 0 ? splits : 1, 0, tiles_t > 1 ? BN : (KIND * n + 7) / 8 * 8};
    if (tile_rows == 0 && splits == 0) {
        long best = -1;
        for (int parts = 1; parts <= 8 && (parts == 1 || 2 * parts <= num_kb); parts *= 2) {
            // alone: tiles of 128 rows, lowered until as many rounds of CTAs as they take are full; clusters of 2, 4 and 8 find room for
            // 148, 132 and 120 CTAs
            const long sms = parts == 4 ? 132 : parts == 8 ? 120 : SMS, per_part = (long)tiles_t * parts, all = (long)(m + 127) / 128 * per_part;
            const long columns = (all + sms - 1) / sms * sms / per_part;
            const int rows = parts > 1 ? 128 : lowered((m + columns - 1) / columns);
            const long ctas = (long)(m + rows - 1) / rows * per_part, each = (ctas + sms - 1) / sms, together = each < 2 ? each : 2;
            const long bytes = (long)(rows * (KIND == CODES ? 136 : 68) * together) / 42, products = 5L * BN * together / 2;
            const long stages = (num_kb + parts - 1) / parts, stage = bytes > products ? bytes : products, x_rows = n < P::TOKENS ? n : P::TOKENS;
            const long cost = (each + 1) / 2 * (2750 + stages * (stage > 350 ? stage : 350) + (parts == 1 ? 80 * x_rows : 0)) +
                              (parts == 1 ? 0 : (parts == 2 ? 1200 : parts == 4 ? 1850 : 5850) + 100 * x_rows);
            if (best < 0 || cost < best) { best = cost; s.tile_rows = rows; s.splits = parts; }
        }
    }
    const int stage = s.tile_rows * 128 + P::B_BYTES + P::SA_BYTES + P::SB_BYTES;
    // a CTA by itself on its SM (4,096 x 4,096 and 64 rows, 128 x 4: 10.2 us, 15.2 with as little as where two share it; eight rows 6.3 and 6.9)
    const int room = (long)(m + s.tile_rows - 1) / s.tile_rows * tiles_t * s.splits <= SMS ? ALONE_SMEM : FEW_SMEM;
    s.stages = (room - 3 * 1024 - (s.splits > 1 ? P::PART * s.tile_rows * 4 : 0)) / stage;
    const int columns = (256 - BN) / P::SCALE_COLS;
    s.stages = s.stages < columns ? s.stages : columns;
    s.stages = s.stages < 16 ? s.stages : 16;
    const int own = (num_kb + s.splits - 1) / s.splits;
    s.stages = s.stages < own ? s.stages : own;
    s.stages = s.stages < 1 ? 1 : s.stages;
    s.tmem_cols = P::tmem_cols(s.stages);
    return s;
}

template <int KIND, int BN, bool INSIDE>
static int launch_few(const void* w, const void* x, int n, int m, int k, Params p, int tile_rows, int splits, cudaStream_t stream) {
    using P = Plan<KIND, BN>;
    const int tiles_t = (n + P::TOKENS - 1) / P::TOKENS;
    if (tiles_t > 65535) return IB_ERR_UNSUPPORTED;
    const Shape sh = shape_for<KIND, BN>(n, m, (k + (KIND == CODES ? 255 : 127)) / (KIND == CODES ? 256 : 128), tiles_t, tile_rows, splits);
    CUtensorMap map_w, map_x;
    if (int r = make_maps<KIND>(&map_w, &map_x, w, x, n, m, k, sh.tile_rows, sh.x_rows, p)) return r;
    if (sh.splits > 8 || sh.splits > p.num_kb || sh.tile_rows % sh.splits) return IB_ERR_ARGUMENT;
    size_t smem = 1024 + (size_t)sh.stages * (sh.tile_rows * 128 + P::B_BYTES + P::SA_BYTES + P::SB_BYTES) +
                  (sh.splits > 1 ? P::PART * sh.tile_rows * 4 : 0) + 16 * sh.stages + 64;
    // the products read 128 rows of A from where the last stage's tile starts, and no less than 128 rows of B are kept readable
    const size_t a_end = 1024 + (size_t)sh.stages * P::B_BYTES + (size_t)(sh.stages - 1) * sh.tile_rows * 128 + A_BYTES;
    const size_t b_end = 1024 + (size_t)(sh.stages - 1) * P::B_BYTES + 128 * 128;
    smem = smem < a_end ? a_end : smem;
    smem = smem < b_end ? b_end : smem;
    // no more CTAs on an SM than have their columns of tensor memory at once: CTAs of clusters that wait for columns could wait
    // for one another
    const size_t alone = (size_t)227 * 1024 / (512 / sh.tmem_cols + 1) + 1;
    smem = smem < alone ? alone : smem;
    static IbDeviceSet done;
    if (int r = ib_allow_dynamic_smem(done, few_rows_kernel<KIND, BN, INSIDE>, 200 * 1024)) return r;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((m + sh.tile_rows - 1) / sh.tile_rows, tiles_t, sh.splits);
    cfg.blockDim = dim3(THREADS + (INSIDE ? 256 : 128));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = sh.splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    // (also behind pieces_kernel, which writes no weights: it lets this kernel start before it has waited itself, and what is ahead of it may write them)
    p.wait_first = !ib_pdl_enabled;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, few_rows_kernel<KIND, BN, INSIDE>, map_w, map_x, p, sh);
    return e == cudaSuccess ? ib_launch_status() : (int)e;
}

template <int KIND, int BN, int STAGES>
static int launch(const void* w, const void* x, int n, int m, int k, Params p, cudaStream_t stream) {
    using P = Plan<KIND, BN>;
    constexpr int SMEM = Many<KIND, BN, STAGES>::SMEM;
    static IbDeviceSet done;
    if (int r = ib_allow_dynamic_smem(done, gemm_kernel<KIND, BN, STAGES>, SMEM)) return r;
    const long tiles = (long)((n + P::TOKENS - 1) / P::TOKENS) * ((m + PAIR * BM - 1) / (PAIR * BM));
    if (tiles > (1 << 30)) return IB_ERR_UNSUPPORTED;
    CUtensorMap map_w, map_x, map_sw, map_sx;
    if (int r = make_maps<KIND>(&map_w, &map_x, w, x, n, m, k, BM, BN / PAIR, p)) return r;
    if (int r = make_scale_map(&map_sw, p.w_scales, p.scale_tiles, (m + BM - 1) / BM, P::K_TILES, 1)) return r;
    if (int r = make_scale_map(&map_sx, p.x_scales, p.scale_tiles, KIND == CODES ? (n + 127) / 128 : (n + P::TOKENS - 1) / P::TOKENS * P::B_GROUPS, P::K_TILES,
                               P::B_GROUPS)) return r;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(PAIR * (tiles < SMS / PAIR ? tiles : SMS / PAIR)));
    cfg.blockDim = dim3(THREADS + 32);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    p.wait_first = !ib_pdl_enabled;      // as in launch_few
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_kernel<KIND, BN, STAGES>, map_w, map_x, map_sw, map_sx, p);
    return e == cudaSuccess ? ib_launch_status() : (int)e;
}

// Tokens of a tile of the product that rows as pieces go through.  17 to 64 float32 rows are several tiles of 16 that read the weights
// again, or one or two of 32 on pairs of CTAs, which want many rows of W (us of 32 rows: 4,096 x 24,576 35 and 21, 4,096 x 4,096 10.3 and 11.6,
// 12,288 x 4,096 17 and 25; 64 rows 45 and 30, 12.7 and 12.8, 26 and 27; between 4,096 and 24,576 rows of W it was not measured).
static int tile_tokens(int x_kind, int n, int m) {
    if (x_kind == 1) return n <= 16 || (n <= 64 && m <= 8192) ? 16 : 32;
    return n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 96;
}
static long pieces_bytes(int parts, int n, int k) { return ((long)parts * n * ((k + 127) / 128 * 128) + 511) / 512 * 512; }

template <typename T, int PARTS>
static int make_pieces(const void* x, long ldx, int n, int k, int tokens, unsigned char* pieces, cudaStream_t stream) {
    const bool one = (long)n * ((k + 255) / 256) <= SMS * 64;
    const dim3 grid(few::strips(n, k, one ? 1 : 2, PIECES_WARPS));
    if (grid.x == 0) return IB_ERR_UNSUPPORTED;
    ib_launch_early(one ? pieces_kernel<T, PARTS, 1> : pieces_kernel<T, PARTS, 2>, grid, dim3(32 * PIECES_WARPS), 0, stream, (const T*)x, ldx, n, k, tokens, (uint2*)pieces,
                    (unsigned*)(pieces + pieces_bytes(PARTS, n, k)));
    return ib_launch_status();
}

}  // namespace mx4

IB_EXPORT int ib_gemm_mx4_error(int reset) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, mx4::g_error, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(mx4::g_error, &zero, sizeof(int));
    }
    return v;
}
IB_EXPORT int ib_gemm_mx4_error_async(int* out, cudaStream_t stream) {
    return (int)cudaMemcpyFromSymbolAsync(out, mx4::g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}

// the bytes of workspace that ib_gemm_mx4 wants: pieces, then their scales (from a multiple of 512 on)
IB_EXPORT long ib_gemm_mx4_workspace(int x_kind, int n, int k) {
    if (x_kind == 2 || (x_kind == 0 && n <= mx4::INSIDE_ROWS)) return 0;
    // (tiles of 32 float32 tokens take the more room)
    const long tokens = mx4::tile_tokens(x_kind, n, 1 << 24), parts = x_kind == 1 ? mx4::PIECES_F32 : mx4::PIECES_BF16;
    const long scale_rows = (n + tokens - 1) / tokens * ((tokens * parts + 127) / 128 * 128);      // whole tiles of tokens
    return mx4::pieces_bytes(x_kind == 1 ? mx4::PIECES_F32 : mx4::PIECES_BF16, n, k) + scale_rows / 128 * few::scale_tiles(k) * 512;
}

// y [n, m] = x w^T.  x_kind 0: bfloat16 rows, 1: float32 rows (both ldx elements apart, `workspace` on 16 bytes), 2: a 4-bit
// matrix (x its codes, x_scales its scales).  tile_rows: rows of w
// a tile of the kernel for few rows (a multiple of 8 up to 128), splits: CTAs that share a tile's K (1, 2, 4, 8); both 0: chosen here.
struct IbGemmMx4 {
    const void *x, *x_scales, *w, *w_scales;
    void *y, *workspace;
    cudaStream_t stream;
    long x_kind, ldx, n, m, k, y_is_f32, ldy, tile_rows, splits;
};
IB_EXPORT int ib_gemm_mx4(const IbGemmMx4* c) {
    using namespace mx4;
    if (c->n > (1 << 24) || c->m > (1 << 24) || c->k > (1 << 24)) return IB_ERR_UNSUPPORTED;
    const void *x = c->x, *x_scales = c->x_scales, *w = c->w, *w_scales = c->w_scales;
    void *y = c->y, *workspace = c->workspace;
    const cudaStream_t stream = c->stream;
    const long ldx = c->ldx, ldy = c->ldy;
    const int x_kind = (int)c->x_kind, n = (int)c->n, m = (int)c->m, k = (int)c->k, y_is_f32 = (int)c->y_is_f32, tile_rows = (int)c->tile_rows,
              splits = (int)c->splits;
    if (n < 0 || m < 0 || k <= 0 || ldy < m || x_kind < 0 || x_kind > 2 || ldx < k || splits < 0 || tile_rows < 0 || tile_rows > 128 || tile_rows % 8) return IB_ERR_ARGUMENT;
    if (n == 0 || m == 0) return IB_OK;
    Params p = {};
    p.y = y;
    p.ldy = ldy;
    p.y_is_f32 = y_is_f32;
    p.y_wide = reinterpret_cast<uintptr_t>(y) % 16 == 0 && ldy * (y_is_f32 ? 4 : 2) % 16 == 0;
    p.n_tok = n;
    p.n_out = m;
    p.x = x;
    p.ldx = ldx;
    p.k = k;
    p.wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * (x_kind ? 4 : 2) % 16 == 0;
    p.w_scales = (const unsigned char*)w_scales;
    if (x_kind == 0 && n <= INSIDE_ROWS) return launch_few<PIECES_BF16, 16, true>(w, nullptr, n, m, k, p, tile_rows, splits, stream);
    if (x_kind == 2) {
        p.x_scales = (const unsigned char*)x_scales;
        if (n <= 16) return launch_few<CODES, 16, false>(w, x, n, m, k, p, tile_rows, splits, stream);
        if (n <= 32) return launch_few<CODES, 32, false>(w, x, n, m, k, p, tile_rows, splits, stream);
        if (n <= 64) return launch_few<CODES, 64, false>(w, x, n, m, k, p, tile_rows, splits, stream);
        return launch<CODES, 192, 5>(w, x, n, m, k, p, stream);
    }
    unsigned char* pieces = (unsigned char*)workspace;
    const int tokens = tile_tokens(x_kind, n, m);
    if (x_kind == 1) {
        p.x_scales = pieces + pieces_bytes(PIECES_F32, n, k);
        if (int r = make_pieces<float, PIECES_F32>(x, ldx, n, k, tokens, pieces, stream)) return r;
        if (tokens == 16) return launch_few<PIECES_F32, 80, false>(w, pieces, n, m, k, p, tile_rows, splits, stream);
        return launch<PIECES_F32, 160, 6>(w, pieces, n, m, k, p, stream);
    }
    p.x_scales = pieces + pieces_bytes(PIECES_BF16, n, k);
    if (int r = make_pieces<__nv_bfloat16, PIECES_BF16>(x, ldx, n, k, tokens, pieces, stream)) return r;
    if (tokens == 16) return launch_few<PIECES_BF16, 32, false>(w, pieces, n, m, k, p, tile_rows, splits, stream);
    if (tokens == 32) return launch_few<PIECES_BF16, 64, false>(w, pieces, n, m, k, p, tile_rows, splits, stream);
    if (tokens == 64) return launch_few<PIECES_BF16, 128, false>(w, pieces, n, m, k, p, tile_rows, splits, stream);
    return launch<PIECES_BF16, 192, 6>(w, pieces, n, m, k, p, stream);
}
