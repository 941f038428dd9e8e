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
// Accumulators are float32 in tensor memory.  Roles: warp 0 copies, warp 1 products, warps 2..5 read back.
//
// With few output tiles K is cut over a cluster (1, 1, splits): every CTA sends its partial sums to their owners (each has
// an equal share of the tile's rows) through distributed shared memory, one cluster barrier follows, and the owner adds
// them in the order of the ranks.  Every wait is bounded and reports through this file's error word.
#include <cuda.h>

#include "few_bits.cuh"
#include "sm100.cuh"

namespace mx4 {

using namespace sm100;

constexpr int BM = 128, THREADS = 192, A_BYTES = BM * 128;
// what a kernel's rows are: the number of pieces of a number, CODES for 4-bit rows
enum { CODES = 1, PIECES_BF16 = 2, PIECES_F32 = 5 };

__device__ int g_error = 0;
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, int code) {
    return mbar_wait_bounded(bar, parity, &g_error, code);
}

struct Params {
    void* y;
    long ldy;
    int y_is_f32, n_tok, n_out, num_kb;      // num_kb: stages that K takes
    const unsigned char *w_scales, *x_scales;
    int scale_tiles;                         // 128-column tiles of scales per 128 rows
};

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_remote_f32(unsigned local_addr, unsigned rank, float v) {
    unsigned remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}
// `bytes` (a multiple of 16) from global to shared memory
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 512 bytes of scales (32 rows of 16 bytes, eight rows 128 bytes apart) into four columns of tensor memory, the same in
// every quarter of the lanes
__device__ __forceinline__ void scales_to_tmem(unsigned tmem, unsigned smem_addr) {
    unsigned long long d = 0;
    d |= (unsigned long long)((smem_addr & 0x3FFFF) >> 4);
    d |= (unsigned long long)(128 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
template <int KIND>
__device__ __forceinline__ void umma_scaled(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa,
                                            unsigned sb, unsigned accumulate) {
    if constexpr (KIND != CODES)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}

// the plan of a kernel's shared and tensor memory
template <int KIND, int BN, int STAGES> struct Plan {
    static constexpr int TOKENS = BN / KIND;                            // of a tile
    static constexpr int B_BYTES = BN * 128;
    static constexpr int K_TILES = KIND != CODES ? 1 : 2;               // 128-column tiles of scales a stage
    static constexpr int B_GROUPS = (BN + 127) / 128;                    // 128-row tiles of scales
    static constexpr int SA_BYTES = 512 * K_TILES, SB_BYTES = 512 * K_TILES * B_GROUPS;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
    static constexpr int SCALE_COLS = 4 * K_TILES * (1 + B_GROUPS);      // of tensor memory a stage
    static constexpr int WANT = BN + STAGES * SCALE_COLS;
    static constexpr int TMEM_COLS = WANT <= 32 ? 32 : WANT <= 64 ? 64 : WANT <= 128 ? 128 : WANT <= 256 ? 256 : 512;
    static_assert(WANT <= 512, "tensor memory");
    static_assert(KIND != PIECES_F32 || BN == 80, "read back sixteen tokens at a time");
    static constexpr bool SPLITS = TOKENS <= 64;                         // K may be cut over a cluster
    static constexpr int RECV_BYTES = SPLITS ? TOKENS * BM * 4 : 0;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE_BYTES + RECV_BYTES + 16 * STAGES + 64 + 1024;
};

template <int KIND, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS) gemm_kernel(const __grid_constant__ CUtensorMap map_w,
                                                       const __grid_constant__ CUtensorMap map_x, const Params p) {
    using P = Plan<KIND, BN, STAGES>;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
    unsigned char* a_tiles = smem;
    unsigned char* b_tiles = a_tiles + STAGES * A_BYTES;
    unsigned char* sa_tiles = b_tiles + STAGES * P::B_BYTES;
    unsigned char* sb_tiles = sa_tiles + STAGES * P::SA_BYTES;
    float* recv = reinterpret_cast<float*>(sb_tiles + STAGES * P::SB_BYTES);     // [rank of the sender][token][rows owned]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(reinterpret_cast<unsigned char*>(recv) + P::RECV_BYTES);
    const unsigned full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), accum = smem_u32(bars + 2 * STAGES);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 2 * STAGES + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_f = blockIdx.x, tile_t = blockIdx.y, splits = gridDim.z;
    const int kb0 = (int)((long)blockIdx.z * p.num_kb / splits), nkb = (int)((long)(blockIdx.z + 1) * p.num_kb / splits) - kb0;   // >= 1

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        mbar_init(accum, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(P::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = *tmem_slot;
    bool ok = true;
    if (P::SPLITS && splits > 1) cluster_arrive();       // "this CTA runs": looked at before the first store to it

    if (warp == 0) {
        if (lane == 0) {
            const unsigned long long pol = policy_evict_first();
            constexpr unsigned W_TX = KIND != CODES ? A_BYTES / 2 : A_BYTES;     // what a tile of weights counts on its barrier
            auto load_w = [&](int i, int s) {
                mbar_expect_tx(full0 + 8 * s, W_TX + P::B_BYTES + P::SA_BYTES + P::SB_BYTES);
                tma_load_2d_hint(smem_u32(a_tiles + s * A_BYTES), &map_w, (kb0 + i) * 128, tile_f * BM, full0 + 8 * s, pol);
                bulk_load(smem_u32(sa_tiles + s * P::SA_BYTES), p.w_scales + ((long)tile_f * p.scale_tiles + (long)(kb0 + i) * P::K_TILES) * 512,
                          P::SA_BYTES, full0 + 8 * s);
            };
            auto load_x = [&](int i, int s) {
                tma_load_2d(smem_u32(b_tiles + s * P::B_BYTES), &map_x, (kb0 + i) * 128, tile_t * BN, full0 + 8 * s);
#pragma unroll
                for (int g = 0; g < P::B_GROUPS; ++g)
                    bulk_load(smem_u32(sb_tiles + s * P::SB_BYTES + g * P::SA_BYTES),
                              p.x_scales + ((long)(tile_t * P::B_GROUPS + g) * p.scale_tiles + (long)(kb0 + i) * P::K_TILES) * 512,
                              P::SA_BYTES, full0 + 8 * s);
            };
            const int head = nkb < STAGES ? nkb : STAGES;    // the first weights are on their way before the kernel ahead is done
            for (int i = 0; i < head; ++i) load_w(i, i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int i = 0; i < head; ++i) load_x(i, i);
            for (int i = head; i < nkb; ++i) {
                const int s = i % STAGES;
                if (!mbar_wait(empty0 + 8 * s, ((i / STAGES) - 1) & 1, 1)) { ok = false; break; }
                load_w(i, s);
                load_x(i, s);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr unsigned FORMATS = KIND != CODES ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);   // e2m1 and e4m3, e2m1 twice
            constexpr unsigned IDESC = FORMATS | ((unsigned)(BN >> 3) << 17) | (1u << 23) | ((unsigned)(BM >> 4) << 24);
            for (int i = 0; i < nkb; ++i) {
                const int s = i % STAGES;
                if (!mbar_wait(full0 + 8 * s, (i / STAGES) & 1, 2)) { ok = false; break; }
                fence_after();
                const unsigned sa = tmem + BN + s * P::SCALE_COLS, sb = sa + 4 * P::K_TILES;
#pragma unroll
                for (int j = 0; j < P::K_TILES; ++j) {
                    scales_to_tmem(sa + 4 * j, smem_u32(sa_tiles + s * P::SA_BYTES + 512 * j));
#pragma unroll
                    for (int g = 0; g < P::B_GROUPS; ++g)     // the column tiles one after the other, the row tiles of each side by side
                        scales_to_tmem(sb + 4 * (j * P::B_GROUPS + g), smem_u32(sb_tiles + s * P::SB_BYTES + g * P::SA_BYTES + 512 * j));
                }
                const unsigned long long da = desc_k_major(smem_u32(a_tiles + s * A_BYTES));
                const unsigned long long db = desc_k_major(smem_u32(b_tiles + s * P::B_BYTES));
#pragma unroll
                for (int k = 0; k < 4; ++k) {                 // 32 bytes of each row: 32 numbers spread to bytes, or 64 packed ones
                    const unsigned tile = KIND != CODES ? 0 : k >> 1, id = KIND != CODES ? k : (k & 1) * 2;
                    umma_scaled<KIND>(tmem, da + 2 * k, db + 2 * k, IDESC | (id << 4) | (id << 29), sa + 4 * tile,
                                      sb + 4 * P::B_GROUPS * tile, (i | k) != 0);
                }
                umma_commit(empty0 + 8 * s);
            }
            umma_commit(accum);
        }
    }

    const int q = warp & 3, row = q * 32 + lane, feature = tile_f * BM + row;
    const unsigned rank = blockIdx.z;
    const int owned = BM / splits;           // rows of the tile that a CTA of the cluster adds up and stores
    const int t0 = tile_t * P::TOKENS, tokens = p.n_tok - t0 < P::TOKENS ? p.n_tok - t0 : P::TOKENS;
    auto store = [&](int t, int f, float v) {
        if (p.y_is_f32) reinterpret_cast<float*>(p.y)[(long)(t0 + t) * p.ldy + f] = v;
        else reinterpret_cast<__nv_bfloat16*>(p.y)[(long)(t0 + t) * p.ldy + f] = __float2bfloat16_rn(v);
    };
    if (P::SPLITS && splits > 1) cluster_wait();
    if (warp >= 2) {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // y may still be read by the kernel ahead
        ok = mbar_wait(accum, 0, 3);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
        if (ok && g_error == 0) {
            constexpr int COLS = KIND == PIECES_F32 ? 80 : 16, STEP = COLS / KIND;     // accumulator columns at a time, their tokens
#pragma unroll 1
            for (int c = 0; c * STEP < tokens; ++c) {
                float v[COLS / 16][16];
#pragma unroll
                for (int i = 0; i < COLS / 16; ++i) tmem_ld16(tmem + ((unsigned)(q * 32) << 16) + COLS * c + 16 * i, v[i]);
#pragma unroll
                for (int j = 0; j < STEP; ++j) {
                    float r = 0.0f;
#pragma unroll
                    for (int i = KIND - 1; i >= 0; --i) r += v[(KIND * j + i) / 16][(KIND * j + i) % 16];
                    const int t = c * STEP + j;
                    if (t >= tokens) break;
                    if (P::SPLITS && splits > 1)
                        st_remote_f32(smem_u32(recv + ((size_t)rank * P::TOKENS + t) * owned + row % owned), (unsigned)(row / owned), r);
                    else if (feature < p.n_out) store(t, feature, r);
                }
            }
        }
    }
    if (P::SPLITS && splits > 1) {
        cluster_arrive();
        cluster_wait();                      // every part of the rows that this CTA owns is in its shared memory
        if (warp >= 2 && g_error == 0) {
            for (int i = (int)threadIdx.x - 64; i < tokens * owned; i += 128) {
                const int t = i / owned, r = i % owned, f = tile_f * BM + (int)rank * owned + r;
                if (f >= p.n_out) continue;
                float sum = 0.0f;
                for (int part = 0; part < splits; ++part) sum += recv[((size_t)part * P::TOKENS + t) * owned + r];
                store(t, f, sum);
            }
        }
    }
    // after a wait that ran out the copies in flight are given time to land before the shared memory is given back
    if (!ok) for (const unsigned long long t = global_ns(); global_ns() - t < 20000000ull;) {}
    fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::TMEM_COLS));
}

// Where the scales of a row's first piece stand: the tiles of 80 columns that five pieces a number take have tiles of 128
// rows of scales of their own; tiles of two pieces a number start where tiles of scales do.
template <int PARTS> __host__ __device__ __forceinline__ int pieces_scale_row(int row) {
    return PARTS == PIECES_F32 ? row / 16 * 128 + row % 16 * PARTS : row * PARTS;
}
// Rows as pieces: row PARTS * t + i of `pieces` [PARTS * n, kp] holds piece i of row t, kp = width rounded up to 128.  A
// thread takes eight numbers, four threads a block of 32, sixteen a word of four scales.
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) pieces_kernel(const T* __restrict__ x, long ldx, int rows, int width, int wide,
                                                     uint2* __restrict__ pieces, unsigned* __restrict__ scales) {
    ib_grid_dependency_sync();
    const int tiles = few::scale_tiles(width), per_row = (width + 127) / 128 * 16;
    const long total = (long)rows * per_row;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (total + 31) / 32 * 32; i += (long)gridDim.x * 256) {
        const bool in = i < total;
        const int row = in ? (int)(i / per_row) : 0, g = (int)(i - (long)row * per_row);
        float v[8];
        few::load8<T>(x + (long)row * ldx + 8 * g, in ? width - 8 * g : 0, wide != 0, v);
        const unsigned m = few::block_largest(v);
        const unsigned byte = few::pieces_byte<PARTS>(m);
        const float by = byte == 255u ? 0.0f : few::scale_reciprocal(byte);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = byte == 255u ? 0.0f : v[j] * by;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const uint2 c = few::take_piece(v);
            unsigned word = (byte == 255u ? 255u : byte - 5u * part) << (8 * (threadIdx.x >> 2 & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            if (in) pieces[((long)row * PARTS + part) * per_row + g] = c;
            if (in && (threadIdx.x & 15) == 0) scales[few::scale_word(pieces_scale_row<PARTS>(row) + part, g >> 4, tiles)] = word;
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

// How many CTAs share a tile's K: as many as run at once (two an SM up to 32 columns of tokens' pieces, one beyond), each
// with at least two stages of it.
static int splits_for(int tiles, int num_kb, int resident) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= 148 * resident && num_kb >= 4 * s) s *= 2;
    return s;
}

template <int KIND, int BN, int STAGES>
static int launch(const void* w, const void* w_scales, const void* x, const void* x_scales, int n, int m, int k, Params p, int splits, cudaStream_t stream) {
    using P = Plan<KIND, BN, STAGES>;
    static IbDeviceSet done;
    if (int r = ib_allow_dynamic_smem(done, gemm_kernel<KIND, BN, STAGES>, P::SMEM)) return r;
    CUtensorMap map_w, map_x;
    const long kp = (long)(k + 127) / 128 * 128;
    int r;
    if (KIND != CODES) {
        if ((r = make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, w, kp, m, kp / 2, 128, BM))) return r;
        if ((r = make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, kp, (long)KIND * n, kp, 128, BN))) return r;
        p.num_kb = (int)(kp / 128);
    } else {
        if ((r = make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, kp / 2, m, kp / 2, 128, BM))) return r;
        if ((r = make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, kp / 2, n, kp / 2, 128, BN))) return r;
        p.num_kb = (int)((kp + 255) / 256);
    }
    p.w_scales = (const unsigned char*)w_scales;
    p.x_scales = (const unsigned char*)x_scales;
    p.scale_tiles = few::scale_tiles(k);
    const int tiles_f = (m + BM - 1) / BM, tiles_t = (n + P::TOKENS - 1) / P::TOKENS;
    if (tiles_t > 65535) return IB_ERR_UNSUPPORTED;
    if (!P::SPLITS || tiles_t > 1) splits = 1;
    else if (splits <= 0) splits = splits_for(tiles_f, p.num_kb, P::SMEM <= 113 * 1024 ? 2 : 1);
    if (splits > 8 || splits > p.num_kb || BM % splits) return IB_ERR_ARGUMENT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles_f, tiles_t, splits);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ib_pdl_enabled ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_kernel<KIND, BN, STAGES>, map_w, map_x, p);
    return e == cudaSuccess ? ib_launch_status() : (int)e;
}

static long pieces_bytes(int parts, int n, int k) { return ((long)parts * n * ((k + 127) / 128 * 128) + 511) / 512 * 512; }

template <typename T, int PARTS>
static int make_pieces(const void* x, long ldx, int n, int k, unsigned char* pieces, unsigned char* scales, cudaStream_t stream) {
    const int wide = (reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * sizeof(T) % 16 == 0) ? 1 : 0;
    const long threads = (long)n * ((k + 127) / 128 * 16), blocks = (threads + 255) / 256;
    ib_launch(pieces_kernel<T, PARTS>, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(256), 0, stream, (const T*)x, ldx, n, k, wide,
              (uint2*)pieces, (unsigned*)scales);
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
    if (x_kind == 2) return 0;
    const long scale_rows = x_kind == 1 ? (n + 15) / 16 * 128L : (2L * n + 255) / 256 * 256;      // whole tiles of tokens
    return mx4::pieces_bytes(x_kind == 1 ? mx4::PIECES_F32 : mx4::PIECES_BF16, n, k) + scale_rows / 128 * few::scale_tiles(k) * 512;
}

// y [n, m] = x w^T.  x_kind 0: bfloat16 rows, 1: float32 rows (both ldx elements apart, `workspace` on 16 bytes), 2: a 4-bit
// matrix (x its codes, x_scales its scales).  splits: CTAs that share a tile's K (0: chosen here; 1, 2, 4, 8).
IB_EXPORT int ib_gemm_mx4(const void* x, int x_kind, long ldx, const void* x_scales, const void* w, const void* w_scales, int n, int m,
                          int k, void* y, int y_is_f32, long ldy, void* workspace, int splits, cudaStream_t stream) {
    using namespace mx4;
    if (n < 0 || m < 0 || k <= 0 || ldy < m || x_kind < 0 || x_kind > 2 || ldx < k || splits < 0) return IB_ERR_ARGUMENT;
    if (n == 0 || m == 0) return IB_OK;
    if (n > (1 << 24) || k > (1 << 24)) return IB_ERR_UNSUPPORTED;
    Params p = {};
    p.y = y;
    p.ldy = ldy;
    p.y_is_f32 = y_is_f32;
    p.n_tok = n;
    p.n_out = m;
    unsigned char* pieces = (unsigned char*)workspace;
    if (x_kind == 0) {
        unsigned char* scales = pieces + pieces_bytes(PIECES_BF16, n, k);
        if (int r = make_pieces<__nv_bfloat16, PIECES_BF16>(x, ldx, n, k, pieces, scales, stream)) return r;
        if (n <= 16) return launch<PIECES_BF16, 32, 4>(w, w_scales, pieces, scales, n, m, k, p, splits, stream);
        if (n <= 32) return launch<PIECES_BF16, 64, 3>(w, w_scales, pieces, scales, n, m, k, p, splits, stream);
        if (n <= 64) return launch<PIECES_BF16, 128, 5>(w, w_scales, pieces, scales, n, m, k, p, splits, stream);
        return launch<PIECES_BF16, 256, 4>(w, w_scales, pieces, scales, n, m, k, p, splits, stream);
    }
    if (x_kind == 1) {
        unsigned char* scales = pieces + pieces_bytes(PIECES_F32, n, k);
        if (int r = make_pieces<float, PIECES_F32>(x, ldx, n, k, pieces, scales, stream)) return r;
        return launch<PIECES_F32, 80, 4>(w, w_scales, pieces, scales, n, m, k, p, splits, stream);
    }
    if (n <= 16) return launch<CODES, 16, 5>(w, w_scales, x, x_scales, n, m, k, p, splits, stream);
    if (n <= 32) return launch<CODES, 32, 4>(w, w_scales, x, x_scales, n, m, k, p, splits, stream);
    if (n <= 64) return launch<CODES, 64, 3>(w, w_scales, x, x_scales, n, m, k, p, splits, stream);
    if (n <= 128) return launch<CODES, 128, 4>(w, w_scales, x, x_scales, n, m, k, p, splits, stream);
    return launch<CODES, 256, 4>(w, w_scales, x, x_scales, n, m, k, p, splits, stream);
}
