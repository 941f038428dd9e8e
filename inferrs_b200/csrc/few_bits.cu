// 4-bit matrices: rows to codes and scales and back.  (The layout is in few_bits.cuh, the product in gemm_mx4.cu.)
#include "few_bits.cuh"

// this library's switch for programmatic dependent launch (see common.cuh)
int ib_pdl_enabled = 0;
IB_EXPORT void ib_few_bits_set_pdl(int on) { ib_pdl_enabled = on; }

namespace few {

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
        const unsigned byte = scale_byte(block_largest(v));
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

static inline int blocks_for(long threads) {
    const long b = (threads + 255) / 256;
    return (int)(b < 148 * 32 ? b : 148 * 32);
}

}  // namespace few

// x [rows, width] (float32 or bfloat16, rows ldx elements apart) to codes and scales
struct IbQuantizeMx4 {
    const void* x;
    void *codes, *scales;
    cudaStream_t stream;
    long x_is_f32, ldx, rows, width;
};
IB_EXPORT int ib_quantize_mx4(const IbQuantizeMx4* q) {
    using namespace few;
    if (q->rows > 0x7FFFFFFF || q->width > (1 << 24)) return IB_ERR_UNSUPPORTED;
    const void* x = q->x;
    void *codes = q->codes, *scales = q->scales;
    const cudaStream_t stream = q->stream;
    const long ldx = q->ldx;
    const int x_is_f32 = (int)q->x_is_f32, rows = (int)q->rows, width = (int)q->width;
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
    if (width > (1 << 24)) return IB_ERR_UNSUPPORTED;
    if (rows == 0) return IB_OK;
    const size_t e = out_is_f32 ? 4 : 2;
    const int wide = (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldo * e) % 16 == 0) ? 1 : 0;
    const dim3 grid(blocks_for((long)rows * ((width + 7) / 8)));
    if (out_is_f32) ib_launch(dequantize_kernel<float>, grid, dim3(256), 0, stream, (const unsigned*)codes, (const unsigned char*)scales, rows, width, wide, (float*)out, ldo);
    else ib_launch(dequantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, (const unsigned*)codes, (const unsigned char*)scales, rows, width, wide, (__nv_bfloat16*)out, ldo);
    return ib_launch_status();
}
