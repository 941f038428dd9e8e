// Numbers in few bits: what the kernels of 4-bit matrices and 8-bit keys and values share.
//
// A 4-bit matrix [rows, width] (sign, two bits of exponent, one of mantissa; a power of two per 32 numbers of a row):
//   codes   byte [row][k / 2], the earlier number in the low half; a row takes 64 bytes per 128 numbers, zeros behind width
//   scales  byte [row / 128][k / 128][row % 32][row / 32 % 4][k / 32 % 4] = exponent + 127 (255: no number at all), an even
//           number of 128-column tiles, zeros behind width.  512 bytes are what the block-scaled product wants beside a
//           tile of 128 rows and 128 columns: copied into tensor memory as they stand.
// 8-bit keys and values: e4m3 codes [page][head][place][dim], a float32 scale per vector [page][head][place].
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

// Kernels of this library are launched while the one ahead still runs, captured or not: they either wait before they read
// anything at all, or are told (wait_first) to do so where the kernels ahead may have written what they would fetch early.
// (Not the attention: its CTAs that start early take the places that its others are to have an SM each in.  Four requests of
// 4,096 keys 14.7 -> 16.6 us.)
template <typename... KArgs, typename... Args>
static inline void ib_launch_early(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

namespace few {

__host__ __device__ __forceinline__ long code_pitch(int width) { return (long)((width + 127) / 128) * 64; }
__host__ __device__ __forceinline__ int scale_tiles(int width) { return (width + 255) / 256 * 2; }
// where the four scales of row `row` and columns 128 t .. 128 t + 127 are
__device__ __forceinline__ long scale_word(int row, int t, int tiles) {
    return ((long)(row >> 7) * tiles + t) * 128 + (row & 31) * 4 + (row >> 5 & 3);
}

// The scale byte of a block from the bits of its largest magnitude: the exponent that puts it into 3.5 .. 7 (up to 7 the
// nearest code, 6, is off by at most a seventh; beyond, the next power of two is nearer).  0 for a block of zeros or of
// numbers too small for any exponent, 255 where there is an infinity or no number.
__device__ __forceinline__ unsigned scale_byte(unsigned largest_bits) {
    const int b = (int)((largest_bits + 0x1FFFFFu) >> 23) - 2;      // (a fraction beyond three quarters carries)
    return largest_bits >= 0x7F800000u ? 255u : (unsigned)max(b, 0);
}
// 2^(byte - 127), and its reciprocal (both exact; bytes of scale_byte: 0 .. 253)
__device__ __forceinline__ float scale_value(unsigned byte) {
    return byte == 255u ? __uint_as_float(0x7FC00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ float scale_reciprocal(unsigned byte) {
    return byte == 254u ? __uint_as_float(0x00400000u) : __uint_as_float((254u - byte) << 23);
}
// eight numbers as codes, nearest with ties to even, beyond 6 as 6; the first in the lowest four bits
__device__ __forceinline__ unsigned codes4x8(float a, float b, float c, float d, float e, float f, float g, float h) {
    unsigned r;
    asm("{\n\t.reg .b8 t, u, v, w;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 u, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 v, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 w, %8, %7;\n\tmov.b32 %0, {t, u, v, w};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f), "f"(g), "f"(h));
    return r;
}
// the values of two codes, the low half of the byte first
__device__ __forceinline__ __half2 values4x2(unsigned byte) {
    unsigned r;
    asm("{\n\t.reg .b8 t, u, v, w;\n\tmov.b32 {t, u, v, w}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(r) : "r"(byte));
    return *reinterpret_cast<const __half2*>(&r);
}

// Eight neighbours of a row as they are stored.  load: those from p on, zeros behind the first n, in pieces as wide as the row's place in
// memory allows (a row that starts on 8, 4 or 2 bytes: 2, 4 or 5 pieces; 1,885 x 6,052 bfloat16 to 4 bits and back on 8 bytes 27 us, number
// by number 49); store: the same back.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p, int n, bool wide = false) {
        const unsigned off = wide ? 0u : (unsigned)reinterpret_cast<uintptr_t>(p) & 15u;
        if (n < 8 || (off & 7u)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
        } else if (off == 0) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float2 a = reinterpret_cast<const float2*>(p)[i]; v[2 * i] = a.x; v[2 * i + 1] = a.y; }
        }
    }
    __device__ __forceinline__ void store(float* p, int n) const {
        const unsigned off = (unsigned)reinterpret_cast<uintptr_t>(p) & 15u;
        if (n < 8 || (off & 7u)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i < n) p[i] = v[i];
        } else if (off == 0) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<float2*>(p)[i] = make_float2(v[2 * i], v[2 * i + 1]);
        }
    }
    // the bits of the largest magnitude
    __device__ __forceinline__ unsigned largest() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        return m;
    }
    __device__ __forceinline__ float operator[](int i) const { return v[i]; }
    __device__ __forceinline__ void set(int i, float a, float b) { v[2 * i] = a; v[2 * i + 1] = b; }      // the i-th pair
};
template <> struct Eight<__nv_bfloat16> {
    unsigned w[4];      // two numbers each
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int n, bool wide = false) {
        const unsigned off = wide ? 0u : (unsigned)reinterpret_cast<uintptr_t>(p) & 15u;
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (2 * i < n ? (unsigned)q[2 * i] : 0u) | (2 * i + 1 < n ? (unsigned)q[2 * i + 1] << 16 : 0u);
        } else if (off == 0) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else if ((off & 7u) == 0) {
            const uint2 a = reinterpret_cast<const uint2*>(p)[0], b = reinterpret_cast<const uint2*>(p)[1];
            w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
        } else if ((off & 3u) == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const unsigned*>(p)[i];
        } else {      // the numbers 1, 3 and 5 start on 4 bytes
            const unsigned first = q[0], last = q[7];
            const unsigned m[3] = {*reinterpret_cast<const unsigned*>(q + 1), *reinterpret_cast<const unsigned*>(q + 3), *reinterpret_cast<const unsigned*>(q + 5)};
            w[0] = __byte_perm(first, m[0], 0x5410);
            w[1] = __byte_perm(m[0], m[1], 0x5432);
            w[2] = __byte_perm(m[1], m[2], 0x5432);
            w[3] = __byte_perm(m[2], last, 0x5432);
        }
    }
    __device__ __forceinline__ void store(__nv_bfloat16* p, int n) const {
        const unsigned off = (unsigned)reinterpret_cast<uintptr_t>(p) & 15u;
        unsigned short* q = reinterpret_cast<unsigned short*>(p);
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i < n) q[i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
        } else if (off == 0) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if ((off & 7u) == 0) {
            reinterpret_cast<uint2*>(p)[0] = make_uint2(w[0], w[1]);
            reinterpret_cast<uint2*>(p)[1] = make_uint2(w[2], w[3]);
        } else if ((off & 3u) == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<unsigned*>(p)[i] = w[i];
        } else {
            q[0] = (unsigned short)w[0];
#pragma unroll
            for (int i = 0; i < 3; ++i) *reinterpret_cast<unsigned*>(q + 1 + 2 * i) = __byte_perm(w[i], w[i + 1], 0x5432);
            q[7] = (unsigned short)(w[3] >> 16);
        }
    }
    __device__ __forceinline__ unsigned largest() const {
        unsigned m = w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return max(m & 0xFFFF0000u, m << 16);
    }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16); }
    __device__ __forceinline__ void set(int i, float a, float b) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(a, b);
        w[i] = *reinterpret_cast<const unsigned*>(&two);
    }
};

// the largest magnitude's bits among four lanes' eight numbers (a block of 32)
__device__ __forceinline__ unsigned block_largest(unsigned mine) {
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
    return max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
}
// The work of a warp whose block takes a strip of 256 columns and `per_warp` rows for each of its warps.
struct Strip {
    int row0, column, g;      // the warp's first row, the lane's first column, its place among a row's groups of eight
    __device__ __forceinline__ Strip(int width, int per_warp) {
        const unsigned columns = (unsigned)(width + 255) / 256, rows = blockIdx.x / columns;
        row0 = (int)(rows * (blockDim.x >> 5) + (threadIdx.x >> 5)) * per_warp;
        g = (int)(blockIdx.x - rows * columns) * 32 + (threadIdx.x & 31);
        column = 8 * g;
    }
};
// blocks of `warps` warps, or 0 where they are more than a grid takes
static inline unsigned strips(long rows, int width, int per_warp, int warps) {
    const long b = (rows + per_warp * warps - 1) / (per_warp * warps) * ((width + 255) / 256);
    return b <= 0x7FFFFFFF ? (unsigned)b : 0u;
}

// ---- 8-bit keys and values ----------------------------------------------------------------------------------------------
// four numbers as e4m3 codes, nearest with ties to even, beyond 448 as 448 (no number stays none)
__device__ __forceinline__ unsigned codes8x4(float a, float b, float c, float d) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    return (unsigned)lo | (unsigned)hi << 16;
}
// two codes (the low half first) as f16 pairs: exact
__device__ __forceinline__ unsigned values8x2(unsigned short c) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
__device__ __forceinline__ float value8(unsigned char c) {
    const unsigned v = values8x2(c);
    return __low2float(*reinterpret_cast<const __half2*>(&v));
}
// A key's scale as the scores meet it: an infinite one is none.  (A sum of products times infinity is + or - infinity where the key's numbers
// are infinities of both signs and zeros times infinity, and the negative one would count as a key that is not seen.)
__device__ __forceinline__ float key_scale(float s) { return fmaf(s, 0.0f, s); }
// Numbers as pieces (see gemm_mx4.cu): the first piece's scale byte of a block from the bits of its largest magnitude (the
// largest then lies in 128 .. 256; every further piece's byte is five less, down to 0), and eight numbers' next piece, in
// whose place 32 times what it leaves of them stays.
template <int PARTS> __device__ __forceinline__ unsigned pieces_byte(unsigned largest_bits) {
    const int e = (int)(largest_bits >> 23);
    return e == 255 ? 255u : (unsigned)max(e - 7, 5 * (PARTS - 1));
}
__device__ __forceinline__ uint2 take_piece(float (&v)[8]) {
    uint2 c;
    c.x = codes8x4(v[0], v[1], v[2], v[3]);
    c.y = codes8x4(v[4], v[5], v[6], v[7]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned two = values8x2((unsigned short)((j < 2 ? c.x : c.y) >> (16 * (j & 1))));
        const float2 taken = __half22float2(*reinterpret_cast<const __half2*>(&two));
        v[2 * j] = 32.0f * (v[2 * j] - taken.x);
        v[2 * j + 1] = 32.0f * (v[2 * j + 1] - taken.y);
    }
    return c;
}
// What a vector with the largest magnitude `a` is multiplied by before its numbers are rounded, and its scale.  0: its codes are
// zeros.  A vector whose numbers are all below 2^-100 counts as zeros; one with an infinity or no number has a scale that is no
// number, and reads back as none (codes that are none would reach, in the attention's products, rows that do not see the vector).
__device__ __forceinline__ void vector_scale(float a, float& by, float& scale) {
    const bool some = a >= 7.888609052210118e-31f, none = !(a <= 3.402823466e38f);
    by = some && !none ? 448.0f / a : 0.0f;
    scale = none ? __uint_as_float(0x7FC00000u) : some ? a / 448.0f : 0.0f;
}

}  // namespace few

// Attention of bfloat16 rows over pages (a multiple of 16 places) of 8-bit keys and values, heads of 64, 128 or 256 numbers.  tile_req null: every row
// is a tile of its own (row_request says whose); else tile i holds up to tile_tokens rows of request tile_req[i] (-1: none)
// from row tile_row0[i] on, and request r's rows end at q_start[r + 1]; tiles of more than 32 (row, head) pairs of a key/value head
// run on attention_kv8_prompt.cu's kernel.  splits: CTAs that share a tile's keys (1, 2, 4, 8, 16; 0: chosen here by max_len, which
// no position is beyond).
struct IbAttentionKv8 {
    const void *q, *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    const int *block_table, *row_request, *positions, *tile_req, *tile_row0, *q_start;
    void* out;
    cudaStream_t stream;
    long max_pages, page_size, n_pages, n_req, n, n_tiles, tile_tokens, n_heads, n_kv, d, span, out_ld, splits, max_len;
    double scale;
};
int ib_kv8_prompt(const IbAttentionKv8* c);
