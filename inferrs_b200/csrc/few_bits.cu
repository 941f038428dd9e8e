// 4-bit matrices: rows to codes and scales and back, and the product that works in 32 bits throughout.
// (The layout is in few_bits.cuh; the tensor cores' product of bfloat16 or 4-bit rows in gemm_mx4.cu.)
#include "few_bits.cuh"

// this library's switch for programmatic dependent launch (see common.cuh)
int ib_pdl_enabled = 0;
IB_EXPORT void ib_few_bits_set_pdl(int on) { ib_pdl_enabled = on; }

namespace few {

template <typename T> __device__ __forceinline__ void load8(const T* p, int n, bool wide, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, int n, bool wide, float (&v)[8]) {
    if (wide && n >= 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, int n, bool wide, float (&v)[8]) {
    if (wide && n >= 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.0f;
    }
}

// Rows to 4 bits.  A thread takes eight numbers, four threads a block of 32, sixteen a word of four scales.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, long ldx, int rows, int width, int wide,
                                                       unsigned* __restrict__ codes, unsigned* __restrict__ scales) {
    ib_grid_dependency_sync();
    const int tiles = scale_tiles(width), per_row = tiles * 16;
    const long pitch = code_pitch(width) / 4, total = (long)rows * per_row;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (total + 31) / 32 * 32; i += (long)gridDim.x * 256) {
        const bool in = i < total;
        const int row = in ? (int)(i / per_row) : 0, g = (int)(i - (long)row * per_row);
        float v[8];
        load8<T>(x + (long)row * ldx + 8 * g, in ? width - 8 * g : 0, wide != 0, v);
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const unsigned byte = scale_byte(m);
        unsigned c = 0;
        if (byte != 255u) {
            const float by = scale_reciprocal(byte);
#pragma unroll
            for (int j = 0; j < 4; ++j) c |= codes2(v[2 * j] * by, v[2 * j + 1] * by) << (8 * j);
        }
        unsigned word = byte << (8 * (threadIdx.x >> 2 & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (in && g < pitch) codes[(long)row * pitch + g] = c;
        if (in && (threadIdx.x & 15) == 0) scales[scale_word(row, g >> 4, tiles)] = word;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                         int rows, int width, int wide, T* __restrict__ out, long ldo) {
    ib_grid_dependency_sync();
    const int tiles = scale_tiles(width), per_row = (width + 7) / 8;
    const long pitch = code_pitch(width) / 4, total = (long)rows * per_row;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const int row = (int)(i / per_row), g = (int)(i - (long)row * per_row);
        const unsigned c = codes[(long)row * pitch + g];
        const float s = scale_value(scales[scale_word(row, g >> 4, tiles) * 4 + (g >> 2 & 3)]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = code_value(c >> (4 * j) & 15u) * s;
        T* o = out + (long)row * ldo + 8 * g;
        if (wide && 8 * g + 8 <= width) {
            if constexpr (sizeof(T) == 2) {
                uint4 w;
                unsigned* p = &w.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    p[j] = *reinterpret_cast<unsigned*>(&b);
                }
                *reinterpret_cast<uint4*>(o) = w;
            } else {
                reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (8 * g + j < width) o[j] = ib_from_float<T>(v[j]);
        }
    }
}

// y[t, f] = sum_k x[t, k] w[f, k] with 32-bit multiply-adds: a warp per feature and 16 rows of x, a lane every 256th
// group of eight k; lanes are added up as a tree.  For float32 rows, and what the faster product does not take.
// CODES: x is a 4-bit matrix too.
constexpr int SLOW_ROWS = 16;
template <typename T, typename O, bool CODES>
__global__ void __launch_bounds__(128) product_kernel(const T* __restrict__ x, long ldx, int wide, const unsigned char* __restrict__ x_scales,
                                                      const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                      int n, int m, int k, O* __restrict__ y, long ldy) {
    ib_grid_dependency_sync();
    const int f = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, t0 = blockIdx.y * SLOW_ROWS;
    if (f >= m) return;
    const int tiles = scale_tiles(k);
    const long pitch = code_pitch(k) / 4;
    float acc[SLOW_ROWS];
#pragma unroll
    for (int t = 0; t < SLOW_ROWS; ++t) acc[t] = 0.0f;
    for (int g = lane; 8 * g < k; g += 32) {
        const unsigned c = codes[(long)f * pitch + g];
        const float s = scale_value(scales[scale_word(f, g >> 4, tiles) * 4 + (g >> 2 & 3)]);
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = code_value(c >> (4 * j) & 15u) * s;
#pragma unroll
        for (int t = 0; t < SLOW_ROWS; ++t) {
            if (t0 + t >= n) break;
            float v[8];
            if constexpr (CODES) {
                const unsigned xc = reinterpret_cast<const unsigned*>(x)[(long)(t0 + t) * pitch + g];
                const float xs = scale_value(x_scales[scale_word(t0 + t, g >> 4, tiles) * 4 + (g >> 2 & 3)]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = code_value(xc >> (4 * j) & 15u) * xs;
            } else {
                load8<T>(x + (long)(t0 + t) * ldx + 8 * g, k - 8 * g, wide != 0, v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[t] = fmaf(v[j], w[j], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < SLOW_ROWS; ++t) {
        if (t0 + t >= n) break;
        const float a = ib_warp_sum(acc[t]);
        if (lane == 0) y[(long)(t0 + t) * ldy + f] = ib_from_float<O>(a);
    }
}

static inline int blocks_for(long threads) {
    const long b = (threads + 255) / 256;
    return (int)(b < 148 * 32 ? b : 148 * 32);
}

}  // namespace few

// x [rows, width] (float32 or bfloat16, rows ldx elements apart) to codes and scales
IB_EXPORT int ib_quantize_mx4(const void* x, int x_is_f32, long ldx, int rows, int width, void* codes, void* scales,
                              cudaStream_t stream) {
    using namespace few;
    if (rows < 0 || width <= 0 || ldx < width) return IB_ERR_ARGUMENT;
    if (rows == 0) return IB_OK;
    const size_t e = x_is_f32 ? 4 : 2;
    const int wide = (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * e) % 16 == 0) ? 1 : 0;
    const dim3 grid(blocks_for((long)rows * scale_tiles(width) * 16));
    if (x_is_f32) ib_launch(quantize_kernel<float>, grid, dim3(256), 0, stream, (const float*)x, ldx, rows, width, wide, (unsigned*)codes, (unsigned*)scales);
    else ib_launch(quantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, (const __nv_bfloat16*)x, ldx, rows, width, wide, (unsigned*)codes, (unsigned*)scales);
    return ib_launch_status();
}

IB_EXPORT int ib_dequantize_mx4(const void* codes, const void* scales, int rows, int width, void* out, int out_is_f32, long ldo,
                                cudaStream_t stream) {
    using namespace few;
    if (rows < 0 || width <= 0 || ldo < width) return IB_ERR_ARGUMENT;
    if (rows == 0) return IB_OK;
    const size_t e = out_is_f32 ? 4 : 2;
    const int wide = (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldo * e) % 16 == 0) ? 1 : 0;
    const dim3 grid(blocks_for((long)rows * ((width + 7) / 8)));
    if (out_is_f32) ib_launch(dequantize_kernel<float>, grid, dim3(256), 0, stream, (const unsigned*)codes, (const unsigned char*)scales, rows, width, wide, (float*)out, ldo);
    else ib_launch(dequantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, (const unsigned*)codes, (const unsigned char*)scales, rows, width, wide, (__nv_bfloat16*)out, ldo);
    return ib_launch_status();
}

// y [n, m] = x w^T in 32 bits.  x_kind: 0 bfloat16, 1 float32, 2 a 4-bit matrix (x its codes, x_scales its scales)
IB_EXPORT int ib_product_mx4(const void* x, int x_kind, long ldx, const void* x_scales, const void* codes, const void* scales,
                             int n, int m, int k, void* y, int y_is_f32, long ldy, cudaStream_t stream) {
    using namespace few;
    if (n < 0 || m < 0 || k <= 0 || x_kind < 0 || x_kind > 2 || ldy < m) return IB_ERR_ARGUMENT;
    if (n == 0 || m == 0) return IB_OK;
    const int blocks_t = (n + SLOW_ROWS - 1) / SLOW_ROWS;
    if (blocks_t > 65535) return IB_ERR_UNSUPPORTED;
    const size_t e = x_kind == 1 ? 4 : 2;
    const int wide = (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * e) % 16 == 0) ? 1 : 0;
    const dim3 grid((m + 3) / 4, blocks_t);
    const unsigned* c = (const unsigned*)codes;
    const unsigned char *s = (const unsigned char*)scales, *xs = (const unsigned char*)x_scales;
#define GO(T, O, C) ib_launch(product_kernel<T, O, C>, grid, dim3(128), 0, stream, (const T*)x, ldx, wide, xs, c, s, n, m, k, (O*)y, ldy)
    if (x_kind == 1) { if (y_is_f32) GO(float, float, false); else GO(float, __nv_bfloat16, false); }
    else if (x_kind == 0) { if (y_is_f32) GO(__nv_bfloat16, float, false); else GO(__nv_bfloat16, __nv_bfloat16, false); }
    else { if (y_is_f32) GO(__nv_bfloat16, float, true); else GO(__nv_bfloat16, __nv_bfloat16, true); }
#undef GO
    return ib_launch_status();
}
