// 4-bit matrices: rows to codes and scales and back.  (The layout is in few_bits.cuh, the product in gemm_mx4.cu.)
#include "few_bits.cuh"

// this library's switch for programmatic dependent launch (see common.cuh)
int ib_pdl_enabled = 0;
IB_EXPORT void ib_few_bits_set_pdl(int on) { ib_pdl_enabled = on; }

namespace few {

// A warp takes 256 columns of four rows: a lane eight numbers of each, four lanes a block of 32.  Memory bounds both kernels: every load of
// the four rows is on its way before the first is used, and no index is divided by anything but once a block.  A matrix of 24,576 x 4,096
// (bfloat16) there and back, 508 MB: 171 us a thread and eight numbers at a time, 92 us now (5.5 TB/s); from cold caches two rows a
// warp 64 and 53 us, four 55 and 47, eight 57 and 45.
constexpr int QUANT_ROWS = 4, QUANT_WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(32 * QUANT_WARPS) quantize_kernel(const T* __restrict__ x, long ldx, int rows, int width, int wide,
                                                                    unsigned* __restrict__ codes, unsigned char* __restrict__ scales) {
    ib_grid_dependency_sync();
    x = ib_after_wait(x);
    const Strip at(width, QUANT_ROWS);
    const int lane = threadIdx.x & 31, tiles = scale_tiles(width);
    const long pitch = code_pitch(width) / 4;
    Eight<T> v[QUANT_ROWS];
#pragma unroll
    for (int r = 0; r < QUANT_ROWS; ++r) {
        const bool in = at.row0 + r < rows;
        v[r].load(x + (long)(in ? at.row0 + r : 0) * ldx + at.column, in ? width - at.column : 0, wide != 0);
    }
#pragma unroll
    for (int r = 0; r < QUANT_ROWS; ++r) {
        const int row = at.row0 + r;
        const unsigned byte = scale_byte(block_largest(v[r].largest()));
        const float by = __uint_as_float((254u - min(byte, 253u)) << 23);
        const unsigned c = codes4x8(v[r][0] * by, v[r][1] * by, v[r][2] * by, v[r][3] * by, v[r][4] * by, v[r][5] * by, v[r][6] * by, v[r][7] * by);
        if (row >= rows) break;
        if (at.g < pitch) codes[(long)row * pitch + at.g] = byte == 255u ? 0u : c;
        if ((lane & 3) == 0) scales[4 * scale_word(row, at.g >> 4, tiles) + (lane >> 2 & 3)] = (unsigned char)byte;
    }
}

template <typename T>
__global__ void __launch_bounds__(32 * QUANT_WARPS) dequantize_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ scales,
                                                         int rows, int width, T* __restrict__ out, long ldo) {
    ib_grid_dependency_sync();
    codes = ib_after_wait(codes);
    scales = ib_after_wait(scales);
    const Strip at(width, QUANT_ROWS);
    const int row0 = at.row0, g = at.g, lane = threadIdx.x & 31, tiles = scale_tiles(width);
    const long pitch = code_pitch(width) / 4;
    unsigned c[QUANT_ROWS], word[QUANT_ROWS];
#pragma unroll
    for (int r = 0; r < QUANT_ROWS; ++r) {
        const bool in = row0 + r < rows && g < pitch;
        c[r] = in ? codes[(long)(row0 + r) * pitch + g] : 0u;
        word[r] = in ? scales[scale_word(row0 + r, g >> 4, tiles)] : 0u;
    }
#pragma unroll
    for (int r = 0; r < QUANT_ROWS; ++r) {
        if (row0 + r >= rows || 8 * g >= width) break;
        const float s = scale_value(word[r] >> (8 * (lane >> 2 & 3)) & 255u);
        Eight<T> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 two = __half22float2(values4x2(c[r] >> (8 * j)));
            v.set(j, two.x * s, two.y * s);
        }
        v.store(out + (long)(row0 + r) * ldo + 8 * g, width - 8 * g);
    }
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
    const int wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * (x_is_f32 ? 4 : 2) % 16 == 0;
    const dim3 grid(strips(rows, width, QUANT_ROWS, QUANT_WARPS));
    if (grid.x == 0) return IB_ERR_UNSUPPORTED;
    if (x_is_f32) ib_launch_early(quantize_kernel<float>, grid, dim3(32 * QUANT_WARPS), 0, stream, (const float*)x, ldx, rows, width, wide, (unsigned*)codes, (unsigned char*)scales);
    else ib_launch_early(quantize_kernel<__nv_bfloat16>, grid, dim3(32 * QUANT_WARPS), 0, stream, (const __nv_bfloat16*)x, ldx, rows, width, wide, (unsigned*)codes, (unsigned char*)scales);
    return ib_launch_status();
}

struct IbDequantizeMx4 {
    const void *codes, *scales;
    void* out;
    cudaStream_t stream;
    long out_is_f32, ldo, rows, width;
};
IB_EXPORT int ib_dequantize_mx4(const IbDequantizeMx4* q) {
    using namespace few;
    if (q->rows > 0x7FFFFFFF || q->width > (1 << 24)) return IB_ERR_UNSUPPORTED;
    const void *codes = q->codes, *scales = q->scales;
    void* out = q->out;
    const cudaStream_t stream = q->stream;
    const long ldo = q->ldo;
    const int out_is_f32 = (int)q->out_is_f32, rows = (int)q->rows, width = (int)q->width;
    if (rows < 0 || width <= 0 || ldo < width) return IB_ERR_ARGUMENT;
    if (rows == 0) return IB_OK;
    const dim3 grid(strips(rows, width, QUANT_ROWS, QUANT_WARPS));
    if (grid.x == 0) return IB_ERR_UNSUPPORTED;
    if (out_is_f32) ib_launch_early(dequantize_kernel<float>, grid, dim3(32 * QUANT_WARPS), 0, stream, (const unsigned*)codes, (const unsigned*)scales, rows, width, (float*)out, ldo);
    else ib_launch_early(dequantize_kernel<__nv_bfloat16>, grid, dim3(32 * QUANT_WARPS), 0, stream, (const unsigned*)codes, (const unsigned*)scales, rows, width, (__nv_bfloat16*)out, ldo);
    return ib_launch_status();
}
