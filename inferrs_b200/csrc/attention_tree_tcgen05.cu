// Attention of drafted tokens on the tensor cores (bfloat16, heads of 64 or 128 numbers); attention_tree.cu says what it computes.
//
// A CTA takes 128 or 256 rows ((token, head of the group) pairs) of one key/value head and one part of the keys, in tiles of 128
// keys.  Two streams of 128 rows take turns on the tensor cores: with more than 128 rows each has rows of its own and both see every tile,
// with up to 128 rows both have the same ones and every other tile, and are joined at the end like the parts of a cluster.
// A stream's tile goes
//   S = Q K^T   128 x 128 in tensor memory, both operands from shared memory;
//   P = 2^(S scale - R), one thread a row, written over S as bfloat16 (its rounding is off by 2^-8 of each p at most, and the sums that
//               divide keep 32 bits); R is a running reference that follows the row's maximum once that is 2^8 beyond it;
//   O += P V    in tensor memory, P from there, V as it lies in its page.
// While one stream's threads compute their P the other's products run.
//
// A tile of 128 keys and values of 128 numbers is 64 KB, 2,900 cycles of an SM's share of the copy bandwidth, and needs 1,100 cycles of
// products and as many of exponentials for every 128 rows.  Keys and values come through a ring of tiles that two warps fill, in the
// order in which the products take them: by TMA, a box for every page, and where pages have an odd size with cp.async, 16 bytes a
// lane.  Where there is no key zeros are written.
//
// What bounds it.  16 trees of 64 over up to 16,384 keys, 32 heads on 8 of 128 (165 to 190 us by the order of the requests, 207 where the power limit
// holds the clock at 1.6 GHz; the bytes alone 90): with 256 rows the tensor cores, whose
// products of 128 x 128 x 16 take 85 to 100 cycles where 64 would do, 3,300 a tile, and 16 us of the join.  8 trees of 16 over 2,048 keys (21.3 us;
// 10.6): memory while the ring runs, on 128 of 148 SMs, and about 10,000 of 38,000 cycles before and behind it.  One tree of 8 over 300
// keys (8.7 us): the chain start, one tile (6,000 cycles), join (5,000), much of it waiting for instructions that run once.  Up to 64 rows standing twice
// among the 128, so that more threads shared the exponentials, gained nothing once a tile's halves were handed over one by one (21.8 us; 16
// trees of 16 over 8,192 keys 135, as it is 123).
//
// What no row sees must not reach it: a product cannot leave a value out, and 0 times infinity is no number.  So the values of tiles that
// some row does not see in full come with cp.async, and the warps that fill the ring look at what they brought, put zeros in the place of those that are
// infinite or no numbers, and the rows that see such a value get it added at the end, from its page.
#include "sm100.cuh"
#include "tree.cuh"

namespace tree_tc {

using namespace sm100;
using namespace tree;
typedef __nv_bfloat16 bf16;

constexpr int ROWS = 128, KEYS = 128;
constexpr int PRODUCERS = 8, N_PRODUCERS = 2, ISSUER = 10, THREADS = 11 * 32;     // warps 0..7: softmax, 8 and 9: the ring, 10: products
constexpr float STEP = 8.0f;          // how far (log2) a row's maximum may outgrow its reference
constexpr int SLICE = 24, MOST_SLICES = 64;      // tiles (see cut_of)
constexpr long MOST_SCRATCH = 256L << 20;        // bytes of all slices' sums (see cut_of)
// Requests that are put in order of their length: every CTA does it for itself, a thread n / 352 times n comparisons.  (In order and as they come, trees
// of 4 over 100 to 2,000 keys, 32 heads on 8: 32 requests 45 and 53 us, 64 78 and 84, 128 136 and 136, 256 315 and 270, 1,024 3,763 and 1,018; trees of
// 16 over 10 to 300 keys: 64 requests 41 and 39, 100 68 and 60, 256 186 and 137.)
constexpr int RANKED = 64;

__device__ int g_error = 0;

__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, int code) {
    return mbar_wait_bounded(bar, parity, &g_error, code);
}

template <int D, int NQ> struct Shape {
    static constexpr int TILE = D / 64 * ROWS * 128;               // bytes of 128 vectors: sub-tiles of 64 numbers, 128 bytes a row
    static constexpr int STAGES = D == 128 ? (NQ == 1 ? 6 : 5) : 8;
    static constexpr int OLD = D + 4;                              // floats between two rows of the sums: 16-byte stores of 8 lanes meet no bank twice
    static constexpr int TILES = (NQ + STAGES) * TILE;
    static constexpr int SUMS = 2 * ROWS * OLD * 4;
    // floats of a slice's sums in the scratch, where a tile has up to `most` rows: o [D / 4][line][4], m and l [line][2], whether it met bad values
    static __host__ __device__ constexpr int lines(int most) { return NQ == 1 ? 2 * most : most; }
    static __host__ __device__ constexpr int slice_sums(int most) { return lines(most) * (D + 2) + 4; }
    static constexpr int SMEM = 232448;                            // all that a CTA may have
    static_assert(1024 + TILES + 256 <= SMEM, "");
    static_assert((NQ == 1 ? SUMS + 4 * ROWS * 4 : 0) + (NQ * ROWS + 8) * (OLD + 4) * 4 <= TILES, "the sums take the place of the tiles");
    static_assert(SUMS + 4 * ROWS * 4 <= TILES, "the CTA's own sums too");
    // One CTA an SM, and no other kernel's that holds tensor memory beside it: a CTA that waits for tensor memory holds up its cluster, which may
    // hold the tensor memory that the other one's cluster waits for.
};

struct Small {                 // what stands behind the tiles
    unsigned long long full[8], empty[8], s_full[2], p_full[2][2], o_full, q_full;
    unsigned tmem;
    int req, lo_min, lo_max, bad_values;
};
static_assert(sizeof(Small) <= 256, "");

__device__ __forceinline__ void cp16(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// an arrival when all that this thread has asked for so far is there (who waits for it needs fence_async before products read it)
__device__ __forceinline__ void cp_arrive(unsigned bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Vectors of D numbers to rows 16 g .. 16 g + 15 of a tile; lanes `from` .. `from` + 15 hold their places among the vectors at `base`
// (-1: zeros)
template <int D>
__device__ __forceinline__ void load_rows(unsigned tile, const bf16* base, int index, int from, int g, int lane) {
    constexpr int CHUNKS = D / 8, STEP_ROWS = 32 / CHUNKS;
    const int c = lane % CHUNKS, sub = lane / CHUNKS;
    const unsigned at = tile + (unsigned)((c >> 3) * (ROWS * 128) + g * 16 * 128);
#pragma unroll
    for (int i = 0; i < 16 / STEP_ROWS; ++i) {
        const int r = i * STEP_ROWS + sub, place = __shfl_sync(0xffffffffu, index, from + r);
        cp16(at + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (long)(place < 0 ? 0 : place) * D + c * 8, place < 0 ? 0 : 16);
    }
}

// Zeros for what is no finite number among what this lane has loaded with load_rows to the g-th 16 rows; true if there was any
template <int D>
__device__ __forceinline__ bool clean_rows(unsigned tile, int g, int lane) {
    constexpr int CHUNKS = D / 8, STEP_ROWS = 32 / CHUNKS;
    const int c = lane % CHUNKS, sub = lane / CHUNKS;
    const unsigned at = tile + (unsigned)((c >> 3) * (ROWS * 128) + g * 16 * 128);
    // bit 15 of a half carries over where all bits of its exponent are set
    auto hits = [](unsigned v) { return ((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
    unsigned v[16 / STEP_ROWS][4], any = 0;
#pragma unroll
    for (int i = 0; i < 16 / STEP_ROWS; ++i) {
        const int r = i * STEP_ROWS + sub;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[i][0]), "=r"(v[i][1]), "=r"(v[i][2]), "=r"(v[i][3])
                     : "r"(at + r * 128 + (((c & 7) ^ (r & 7)) << 4)) : "memory");
    }
#pragma unroll
    for (int i = 0; i < 16 / STEP_ROWS; ++i) any |= hits(v[i][0]) | hits(v[i][1]) | hits(v[i][2]) | hits(v[i][3]);
    if (any) {
#pragma unroll 1
        for (int i = 0; i < 16 / STEP_ROWS; ++i) {
            const int r = i * STEP_ROWS + sub;
            const unsigned a = at + r * 128 + (((c & 7) ^ (r & 7)) << 4);
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
                unsigned x;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(a + 4 * k) : "memory");
                x &= ~((hits(x) >> 15) * 0xffffu);
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(a + 4 * k), "r"(x) : "memory");
            }
        }
    }
    return any != 0;
}

// Columns of this warp's lanes of tensor memory, and the wait for them: in one piece, since the compiler may put registers aside
// between the two, before they hold what was asked for
__device__ __forceinline__ void tmem_ld64(unsigned taddr, unsigned (&r)[64]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29"
                 ",%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%"
                 "57,%58,%59,%60,%61,%62,%63}"
                 ", [%64];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(unsigned taddr, unsigned (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29"
                 ",%30,%31}"
                 ", [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// two neighbouring numbers at once
typedef unsigned long long u64;
__device__ __forceinline__ u64 pair(float a, float b) {
    u64 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void apart(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// One lane of the warp, the same every time
__device__ __forceinline__ bool elected() {
    unsigned r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// operand descriptors: desc_k_major and desc_mn_major (groups of 64 numbers ROWS * 128 bytes apart) of sm100.cuh, from the address in 16 bytes
__device__ __forceinline__ u64 words(unsigned lo, unsigned hi) {
    u64 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
constexpr unsigned K_HI = (unsigned)(1024 >> 4) | 1u << 14 | 2u << 29, V_HI = K_HI, K_LO = 1u << 16, V_LO = (unsigned)(ROWS * 128 >> 4) << 16;

struct Place {
    const int* bt;
    int head, keys;
};
__device__ __forceinline__ int key_index(const Args& A, const Place& p, int j) {
    if (j >= p.keys) return -1;
    const int slot = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size;
    const int page = p.bt[slot];
    if (page < 0 || page >= A.n_pages) return -1;
    return (page * A.n_kv + p.head) * A.page_size + (j - slot * A.page_size);
}

// those of the 32 keys from j on whose bit is set and whose page is there
__device__ __noinline__ unsigned with_page(const Args& A, const Place p, int j, unsigned bits) {
#pragma unroll 1
    for (unsigned left = bits; left; left &= left - 1)
        if (key_index(A, p, j + __ffs(left) - 1) < 0) bits &= ~(left & -left);
    return bits;
}

// which of the 32 N keys from jb on a row sees; lo: the first key of the context that it sees
template <int N>
__device__ __forceinline__ void visible(const Args& A, const Span& S, const Place& p, const int* row_words, int lo, int jb, bool bad_pages,
                                        unsigned (&see)[N]) {
    const int first = jb - S.context, at = first >> 5, shift = first & 31;        // (rounds down)
    unsigned w[N + 1];
#pragma unroll
    for (int c = 0; c <= N; ++c) w[c] = at + c >= 0 && at + c < A.words ? (unsigned)row_words[at + c] : 0u;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const int j = jb + 32 * c, a = max(lo - j, 0), b = min(S.context - j, 32), left = S.keys - j;
        unsigned bits = b > a ? (b == 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u) : 0u;
        if (b < 32) {              // (a drafted token behind the tree's last one is behind the keys too)
            const unsigned drafted = __funnelshift_r(w[c], w[c + 1], shift);
            bits |= left >= 32 ? drafted : left > 0 ? drafted & ((1u << left) - 1u) : 0u;
        }
        see[c] = bits;
    }
    if (bad_pages) {               // (rare, and long if it were unrolled: code that is fetched costs time even where it is not run)
#pragma unroll
        for (int c = 0; c < N; ++c) see[c] = with_page(A, p, jb + 32 * c, see[c]);
    }
}

__device__ __forceinline__ void remote_store(unsigned to, const float4& v) {      // into a CTA of the cluster (see ib_cluster_address)
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// A row's numbers e .. e + 3 with the infinite values and no numbers that it sees in tiles that not all rows see
template <int D>
__device__ __noinline__ float4 with_bad_values(const Args& A, const Span S, const Place place, float4 o, int token, int e, int t_first,
                                               int n_tiles, int lo_max) {
    const int lo = first_key(A, S, token);
    const int* words = A.seen + (long)(S.row0 + token) * A.words;
    float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll 1
    for (int t = t_first; t < t_first + n_tiles; ++t) {
        if (!(t * KEYS < lo_max || (t + 1) * KEYS > S.context)) continue;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            unsigned see[1];
            visible(A, S, place, words, lo, t * KEYS + 32 * c, true, see);
            for (; see[0]; see[0] &= see[0] - 1) {
                const bf16* x = static_cast<const bf16*>(A.v) + (long)key_index(A, place, t * KEYS + 32 * c + __ffs(see[0]) - 1) * D + e;
                for (int k = 0; k < 4; ++k) {
                    const float add = __bfloat162float(x[k]);
                    if (!(fabsf(add) < INFINITY)) v[k] += add;
                }
            }
        }
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

// The sum (m, l, the numbers at x and every 32 behind them) joins a row's (top, total, o).  (A sum whose l is 0 is not there: what stands in its
// place is not used.)
template <int QUADS>
__device__ __forceinline__ void join(float& top, float& total, float4 (&o)[QUADS], float m, float l, const float* x, int step = 32) {
    if (l == 0.0f) return;
    float4 v[QUADS];
#pragma unroll
    for (int k = 0; k < QUADS; ++k) v[k] = *reinterpret_cast<const float4*>(x + k * step);
    const float to = fmaxf(top, m), ref = to == -INFINITY ? 0.0f : to, a = ex2(top - ref), b = ex2(m - ref);
    total = fmaf(l, b, total * a);
    top = to;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
        o[k].x = fmaf(v[k].x, b, o[k].x * a); o[k].y = fmaf(v[k].y, b, o[k].y * a);
        o[k].z = fmaf(v[k].z, b, o[k].z * a); o[k].w = fmaf(v[k].w, b, o[k].w * a);
    }
}

// numbers e .. e + 3 of a row (counted token by token), and every `step` behind them, to their place
template <int D, int QUADS>
__device__ __forceinline__ void write_row(const Args& A, const Span& S, const Place& place, int at, int head, int e, int step, float4 (&o)[QUADS],
                                          float total, bool bad_values, int t_first, int n_tiles, int lo_max) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int group = A.group, token = A.group_shift >= 0 ? at >> A.group_shift : at / group;
    bf16* dst = static_cast<bf16*>(A.out) + (long)(S.row0 + token) * A.out_ld + (long)(head * group + at - token * group) * D + e;
    const bool wide = ((unsigned)reinterpret_cast<uintptr_t>(A.out) | (unsigned)A.out_ld * 2) % 8 == 0;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
        float4 v = make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv);
        if (bad_values) v = with_bad_values<D>(A, S, place, v, token, e + k * step, t_first, n_tiles, lo_max);
        if (wide) {
            *reinterpret_cast<uint2*>(dst + k * step) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        } else {
            bf16* to = dst + k * step;
            to[0] = __float2bfloat16_rn(v.x); to[1] = __float2bfloat16_rn(v.y); to[2] = __float2bfloat16_rn(v.z); to[3] = __float2bfloat16_rn(v.w);
        }
    }
}

// In how many slices a request's tiles are cut where there may be `most`: of SLICE tiles or more
__device__ __forceinline__ int slices_of(int tiles, int most) {
    const int n = (tiles + SLICE - 1) / SLICE;
    return n < 1 ? 1 : n > most ? most : n;
}

template <int D, int NQ>
__global__ void __launch_bounds__(THREADS, 1) tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                          const __grid_constant__ Args A, int slices, int ranked, int box,
                                                          float* scratch, int slice_rows) {
    typedef Shape<D, NQ> Sh;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    float* sums = reinterpret_cast<float*>(smem);                 // [2][ROWS][OLD], once the tiles have been used
    float* part_m = reinterpret_cast<float*>(smem + Sh::SUMS);    // [2][ROWS]
    float* part_l = part_m + 2 * ROWS;
    Small& sm = *reinterpret_cast<Small*>(smem + Sh::TILES);
    const unsigned sq = smem_u32(smem), ring = sq + NQ * Sh::TILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (threadIdx.x == PRODUCERS * 32 && box > 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    // `slices` CTAs for the same rows: a cluster whose CTAs take a part of the keys each, or, with a scratch, as many as the keys need
    int unit = blockIdx.x / slices;
    const int part = blockIdx.x - unit * slices;
    const int head = unit % A.n_kv;
    unit /= A.n_kv;
    const int row_tile = unit % A.tiles_of_rows;
    int req = unit / A.tiles_of_rows;
    if (ranked) {                     // the longest contexts first: the grid's last CTAs are short ones
        int* lengths = reinterpret_cast<int*>(smem);
#pragma unroll 1
        for (int i = tid; i < A.n_requests; i += THREADS) lengths[i] = A.context[i];
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < A.n_requests; i += THREADS) {
            const int mine = lengths[i];
            int ahead = 0;
#pragma unroll 4
            for (int j = 0; j < A.n_requests; ++j) ahead += lengths[j] > mine || (lengths[j] == mine && j < i);
            if (ahead == req) sm.req = i;
        }
        __syncthreads();
        req = sm.req;
    }
    const Span S = span_of(A, req);
    const int group = A.group;
    const int first_row = row_tile * (NQ * ROWS);
    const int rows = min(S.n_tree * group - first_row, slice_rows);      // (NQ * ROWS, or what the scratch has room for)
    if (rows <= 0) return;            // (the whole cluster leaves)

    if (tid == 0) {
        sm.lo_min = 0x7fffffff;
        sm.lo_max = 0;
        sm.bad_values = 0;
    }
    // the first keys that the CTA's rows see: the least and the greatest
    auto first_keys = [&]() {
        const int t0 = first_row / group, t1 = (first_row + rows - 1) / group;
#pragma unroll 1
        for (int t = t0 + tid; t <= t1; t += THREADS) {
            const int lo = first_key(A, S, t);
            atomicMin(&sm.lo_min, lo);
            atomicMax(&sm.lo_max, lo);
        }
        __syncthreads();
    };
    if (scratch != nullptr) {
        // A CTA that no slice is left for has no rows to write and no place for sums: it leaves before it takes anything.  What is left behind a
        // span's first keys may be fewer slices than the request's keys alone would give, one even.
        if (A.span != 0) {
            __syncthreads();
            first_keys();
        }
        const int t0 = A.span != 0 ? min(sm.lo_min, S.context) / KEYS : 0;
        if (part >= slices_of((S.keys + KEYS - 1) / KEYS - t0, slices)) return;
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == PRODUCERS && lane == 0) {
#pragma unroll 1
        for (int i = 0; i < Sh::STAGES; ++i) { mbar_init(smem_u32(&sm.full[i]), 32 * N_PRODUCERS); mbar_init(smem_u32(&sm.empty[i]), 1); }
#pragma unroll 1
        for (int g = 0; g < 2; ++g) {
            const int used = NQ == 2 ? rows - g * ROWS : rows;
            mbar_init(smem_u32(&sm.s_full[g]), 1);
            for (int h = 0; h < 2; ++h) mbar_init(smem_u32(&sm.p_full[g][h]), used <= 0 ? 1 : used >= ROWS ? 4 : (used + 31) / 32);
        }
        mbar_init(smem_u32(&sm.o_full), 1);
        mbar_init(smem_u32(&sm.q_full), 256);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (A.span != 0 && scratch == nullptr) first_keys();
    const int lo_min = A.span != 0 ? min(sm.lo_min, S.context) : 0, lo_max = A.span != 0 ? sm.lo_max : 0;
    const unsigned tmem = sm.tmem;
    const int t_first = lo_min / KEYS, all_tiles = (S.keys + KEYS - 1) / KEYS - t_first;
    const int parts = scratch != nullptr ? slices_of(all_tiles, slices) : slices;
    const int t_begin = t_first + all_tiles * part / parts, t_end = t_first + all_tiles * (part + 1) / parts;      // (fewer than 2^24 tiles)
    const int n = t_end - t_begin;
    // tiles that each stream takes
    const int count0 = NQ == 2 ? n : (n + 1) / 2, count1 = NQ == 2 ? (rows > ROWS ? n : 0) : n / 2;
    const Place place = {A.table + (long)req * A.max_pages, head, S.keys};
    // what the cluster's CTAs send this one: `most` rows of each (their sums; references, denominators and whether they met bad values).  With 128
    // rows it lies behind the CTA's own sums.
    const int most = (rows + parts - 1) / parts, over = 65536 / parts + 1;
    auto share_of = [&](int row) { return row * over >> 16; };        // row / parts, for rows below 256 and up to eight parts
    float* inbox = NQ == 1 ? part_l + 2 * ROWS : sums;
    float* inbox_ml = inbox + parts * most * Sh::OLD;
    // keys that some row does not see
    auto partly = [&](int t) { return t * KEYS < lo_max || (t + 1) * KEYS > S.context; };
    bool ok = true;

    if (warp >= PRODUCERS && warp < PRODUCERS + N_PRODUCERS) {
        const int w = warp - PRODUCERS;
        // the ring's entries in the order of the products: with two sets of rows K0 V0 K1 V1 .., else K0 K1 V0 K2 V1 .. V(n-1)
        auto tile_of = [&](int e, bool& values) -> int {
            if (NQ == 2) {
                values = e & 1;
                return e >> 1;
            }
            values = e != 0 && (e == 2 * n - 1 || (e & 1) == 0);
            if (e == 2 * n - 1) return n - 1;
            return e == 0 ? 0 : (e & 1) ? (e + 1) >> 1 : (e - 2) >> 1;
        };
        const int beyond = A.n_pages * A.n_kv * A.page_size;          // a box that starts here is zeros
        auto in_boxes = [&](int t, bool values) { return box > 0 && !(values && partly(t)); };
        // An entry's places: of the box that this lane brings, or of two rows.  They are looked up an entry ahead: the table's answer takes a while.
        int index[2], index_next[2];
        auto look_up = [&](int e, int (&to)[2]) {
            to[0] = to[1] = -1;
            if (e >= 2 * n) return;
            bool values;
            const int t = t_begin + tile_of(e, values), j = t * KEYS;
            if (in_boxes(t, values)) {
                if (lane * box < KEYS) to[0] = key_index(A, place, j + lane * box);
                if (to[0] < 0) to[0] = beyond;
            } else {
                to[0] = key_index(A, place, j + w * 64 + lane);
                to[1] = key_index(A, place, j + w * 64 + 32 + lane);
            }
        };
        look_up(0, index_next);
        int slot = 0, turn = 0;
        for (int e = 0; e < 2 * n; ++e) {
            if (turn > 0 && !mbar_wait(smem_u32(&sm.empty[slot]), (turn - 1) & 1, 1)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            bool values;
            const int t = t_begin + tile_of(e, values);
            index[0] = index_next[0];
            index[1] = index_next[1];
            look_up(e + 1, index_next);
            const unsigned dst = ring + slot * Sh::TILE, full = smem_u32(&sm.full[slot]);
            if (in_boxes(t, values)) {
                // one warp a sub-tile of 64 numbers, one lane a box
                if (lane == 0 && w < D / 64) mbar_expect_tx(full, ROWS * 128);
                else mbar_arrive(full);
                __syncwarp();
                if (lane * box < KEYS && w < D / 64)
                    tma_load_2d(dst + w * (ROWS * 128) + lane * box * 128, values ? &map_v : &map_k, w * 64, index[0], full);
            } else {
#pragma unroll 1
                for (int h = 0; h < 4; ++h)
                    load_rows<D>(dst, static_cast<const bf16*>(values ? A.v : A.k), h < 2 ? index[0] : index[1], 16 * (h & 1), w * 4 + h, lane);
                if (values && partly(t)) {
                    cp_wait_all();
#pragma unroll 1
                    for (int h = 0; h < 4; ++h)
                        if (clean_rows<D>(dst, w * 4 + h, lane)) sm.bad_values = 1;
                    mbar_arrive(full);
                } else {
                    cp_arrive(full);
                }
            }
            if (++slot == Sh::STAGES) { slot = 0; ++turn; }
        }
        cp_wait_all();
    } else if (warp == ISSUER) {
        // the warp runs its loops as a whole, so that addresses and descriptors are the same for all lanes; one lane issues
        constexpr unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(ROWS >> 4) << 24);
        constexpr unsigned idesc_s = idesc | ((unsigned)(KEYS >> 3) << 17), idesc_o = idesc | (1u << 16) | ((unsigned)(D >> 3) << 17);
        const bool leader = elected();
        // (an address of a cluster's CTA has its rank above the 18 bits that a descriptor takes)
        const unsigned ring0 = __shfl_sync(0xffffffffu, (ring & 0x3FFFF) >> 4, 0), q0 = __shfl_sync(0xffffffffu, (sq & 0x3FFFF) >> 4, 0);
        const unsigned tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int last = NQ == 2 && count1 > 0 ? 1 : 0;            // with two sets of rows: the stream that is done with a tile last
        struct Turn { int slot; unsigned phase; };
        Turn k_at = {0, 0}, v_at = {0, 0};                         // the next keys and values: places in the ring
        auto step = [&](Turn& u, int by) {
            u.slot += by;
            if (u.slot >= Sh::STAGES) { u.slot -= Sh::STAGES; u.phase ^= 1; }
        };
        step(v_at, NQ == 2 ? 1 : n == 1 ? 1 : 2);
        auto arrived = [&](const Turn& u) {
            if (!mbar_wait(smem_u32(&sm.full[u.slot]), u.phase, 2)) return false;
            fence_async();
            fence_after();
            return true;
        };
        auto scores = [&](int g) {
            if (!arrived(k_at)) return false;
            if (leader) {
                const unsigned k = ring0 + k_at.slot * (Sh::TILE >> 4), rows_q = q0 + (NQ == 2 ? g * (Sh::TILE >> 4) : 0);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    const unsigned off = ((s >> 2) * (ROWS * 128) + (s & 3) * 32) >> 4;
                    umma(tm + g * 128, words(rows_q + off + K_LO, K_HI), words(k + off + K_LO, K_HI), idesc_s, s != 0);
                }
                umma_commit(smem_u32(&sm.s_full[g]));
                if (NQ == 1 || g == last) umma_commit(smem_u32(&sm.empty[k_at.slot]));
            }
            return true;
        };
        ok = mbar_wait(smem_u32(&sm.q_full), 0, 3);
        // keys: K0 [V0] K1 [V1] .. with two sets of rows; K0 K1 [V0] K2 [V1] .. else.  Values likewise, the last one behind the one before it.
        int k_next = 0, v_next = 0;
        auto k_done = [&]() { step(k_at, NQ == 2 ? 2 : k_next == 0 ? 1 : 2); ++k_next; };
        auto v_done = [&]() { step(v_at, NQ == 2 ? 2 : v_next + 2 < n ? 2 : 1); ++v_next; };
        for (int g = 0; g < 2 && ok; ++g)
            if ((g ? count1 : count0) > 0) {
                ok = scores(g);
                if (NQ == 1 || g == last) k_done();
            }
        for (int i = 0; i < count0 && ok; ++i) {
            for (int g = 0; g < 2 && ok; ++g) {
                if (i >= (g ? count1 : count0)) continue;
                // the products with the first half's P run while the threads make the second half's
                const unsigned v = ring0 + v_at.slot * (Sh::TILE >> 4);
                if (!mbar_wait(smem_u32(&sm.p_full[g][0]), i & 1, 4) || !arrived(v_at)) { ok = false; break; }
                if (leader) {
#pragma unroll
                    for (int s = 0; s < KEYS / 32; ++s)
                        umma_ts(tm + 256 + g * 128, tm + g * 128 + s * 8, words(v + s * (16 * 128 >> 4) + V_LO, V_HI), idesc_o, (i | s) != 0);
                }
                if (!mbar_wait(smem_u32(&sm.p_full[g][1]), i & 1, 4)) { ok = false; break; }
                fence_after();
                if (leader) {
#pragma unroll
                    for (int s = KEYS / 32; s < KEYS / 16; ++s)
                        umma_ts(tm + 256 + g * 128, tm + g * 128 + s * 8, words(v + s * (16 * 128 >> 4) + V_LO, V_HI), idesc_o, (i | s) != 0);
                    if (NQ == 1 || g == last) umma_commit(smem_u32(&sm.empty[v_at.slot]));
                }
                if (NQ == 1 || g == last) v_done();
                if (i + 1 < (g ? count1 : count0)) {
                    ok = scores(g);
                    if (NQ == 1 || g == last) k_done();
                }
            }
        }
        if (leader) umma_commit(smem_u32(&sm.o_full));
        __syncwarp();
    } else {
        // the queries: 16 rows a warp and set
#pragma unroll
        for (int s = 0; s < NQ; ++s) {
            const int r = s * ROWS + warp * 16 + (lane & 15), at = first_row + r, token = at / group;
            const int index = r < rows ? (S.row0 + token) * A.n_heads + head * group + at - token * group : -1;
            load_rows<D>(sq + s * Sh::TILE, static_cast<const bf16*>(A.q), index, 0, warp, lane);
        }
        cp_arrive(smem_u32(&sm.q_full));
        const int g = warp >> 2, r = (warp & 3) * 32 + lane;
        const int used = NQ == 2 ? min(rows - g * ROWS, ROWS) : rows, count = g ? count1 : count0;
        if ((warp & 3) * 32 < used) {
            const bool mine = r < used;
            const int at = first_row + (NQ == 2 ? g * ROWS : 0) + (mine ? r : 0), token = at / group;
            const int lo = first_key(A, S, token);
            const int* words = A.seen + (long)(S.row0 + token) * A.words;
            // a page of the part's keys that is not there: such keys are none (all of the stream's warps look, each for itself)
            bool bad = false;
            if (n > 0) {
                const int j0 = max(t_begin * KEYS, lo_min), j1 = min(t_end * KEYS, S.keys);
#pragma unroll 1
                for (int slot = A.page_shift >= 0 ? (j0 >> A.page_shift) + lane : j0 / A.page_size + lane; (long)slot * A.page_size < j1; slot += 32) {
                    const int page = place.bt[slot];
                    if (page < 0 || page >= A.n_pages) bad = true;
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
            const unsigned s_at = tmem + lanes + g * 128, o_at = tmem + lanes + 256 + g * 128;
            float m = -INFINITY, l = 0.0f;
            for (int i = 0; i < count; ++i) {
                const int t = t_begin + (NQ == 2 ? i : 2 * i + g), j0 = t * KEYS;
                const bool plain = __all_sync(0xffffffffu, !bad && j0 >= lo && j0 + KEYS <= S.context);
                unsigned see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                if (!plain) visible(A, S, place, words, lo, j0, bad, see);
                if (!mbar_wait(smem_u32(&sm.s_full[g]), i & 1, 5)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                // 128 scores and what else a thread keeps are more than its registers: half of them stay, half come twice
                auto hide = [&](auto& x, int at, int c) {
                    if (!plain) {
                        const unsigned bits = c == 0 ? see[0] : c == 1 ? see[1] : c == 2 ? see[2] : see[3];
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(bits >> k & 1u)) x[at + k] = 0xff800000u;
                    }
                };
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto look = [&](const auto& x, int at) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            top4[c] = max3(top4[c], __uint_as_float(x[at + k + 2 * c]), __uint_as_float(x[at + k + 2 * c + 1]));
                };
                unsigned x[64];
                tmem_ld64(s_at, x);
                hide(x, 0, 0);
                hide(x, 32, 1);
                look(x, 0);
                look(x, 32);
                unsigned y[32];
                tmem_ld32(s_at + 64, y);
                hide(y, 0, 2);
                look(y, 0);
                tmem_ld32(s_at + 96, y);
                hide(y, 0, 3);
                look(y, 0);
                const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * A.scale_log2;     // (the scale is positive)
                const bool move = top > m + STEP || (m == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float c = move ? (m == -INFINITY ? 0.0f : ex2(m - top)) : 1.0f;
                    __syncwarp();
                    if (i > 0) {      // (the stream's products are done: the one that gave S came behind them)
#pragma unroll 1
                        for (int e = 0; e < D; e += 32) {
                            unsigned x[32];
                            tmem_ld32(o_at + e, x);
#pragma unroll
                            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * c);
                            tmem_st32(o_at + e, x);
                        }
                        tmem_st_wait();
                    }
                    l *= c;
                    if (move) m = top;
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                const u64 factor = pair(A.scale_log2, A.scale_log2), less = pair(-ref, -ref);
                u64 add[2] = {0, 0};
                auto weigh = [&](const unsigned* x, int c) {
                    unsigned p[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float a, b;
                        apart(fma2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), factor, less), a, b);
                        a = ex2(a);
                        b = ex2(b);
                        add[k & 1] = add2(add[k & 1], pair(a, b));
                        p[k] = pack_bf16(a, b);
                    }
                    tmem_st16(s_at + 16 * c, p);
                };
                weigh(x, 0);
                weigh(x + 32, 1);
                auto hand_over = [&](int h) {
                    tmem_st_wait();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[g][h]));
                    __syncwarp();
                };
                hand_over(0);
                tmem_ld64(s_at + 64, x);
                hide(x, 0, 2);
                hide(x, 32, 3);
                weigh(x, 2);
                weigh(x + 32, 3);
                float a, b;
                apart(add2(add[0], add[1]), a, b);
                l += a + b;
                hand_over(1);
            }
            if (!mbar_wait(smem_u32(&sm.o_full), 0, 6)) ok = false;       // every product is done: the tiles' memory is free
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            if (scratch == nullptr && parts > 1) ib_cluster_sync();          // the cluster's tiles are free: sums may go to any CTA
            if (NQ == 2 && parts == 1 && !sm.bad_values) {
                // no other sums of these rows: they go out from here, a thread a row
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                bf16* dst = static_cast<bf16*>(A.out) + (long)(S.row0 + token) * A.out_ld + (long)(head * group + at - token * group) * D;
                const bool wide = ((unsigned)reinterpret_cast<uintptr_t>(A.out) | (unsigned)A.out_ld * 2) % 16 == 0;
#pragma unroll 1
                for (int e = 0; e < D; e += 32) {
                    unsigned x[32];
                    __syncwarp();      // rows of no token skip the stores
                    tmem_ld32(o_at + e, x);
                    if (!ok || !mine) continue;
                    unsigned y[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float a = count > 0 ? __uint_as_float(x[2 * k]) * inv : 0.0f, b = count > 0 ? __uint_as_float(x[2 * k + 1]) * inv : 0.0f;
                        y[k] = pack_bf16(a, b);
                    }
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        if (wide) {
                            *reinterpret_cast<uint4*>(dst + e + 2 * k) = make_uint4(y[k], y[k + 1], y[k + 2], y[k + 3]);
                        } else {
                            for (int i = 0; i < 4; ++i) {
                                reinterpret_cast<unsigned short*>(dst)[e + 2 * (k + i)] = (unsigned short)y[k + i];
                                reinterpret_cast<unsigned short*>(dst)[e + 2 * (k + i) + 1] = (unsigned short)(y[k + i] >> 16);
                            }
                        }
                    }
                }
            } else if (scratch != nullptr && parts > 1) {
                // the sums of a slice, numbers four by four, so that a warp's stores lie side by side
                float* to = scratch + (((long)(req * A.tiles_of_rows + row_tile) * A.n_kv + head) * slices + part) * Sh::slice_sums(slice_rows);
                const int lines = Sh::lines(slice_rows), all = g * (NQ == 2 ? ROWS : slice_rows) + r;
#pragma unroll 1
                for (int e = 0; e < D && count > 0; e += 32) {
                    unsigned x[32];
                    tmem_ld32(o_at + e, x);
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<uint4*>(to + ((e + k) / 4 * lines + all) * 4) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                }
                *reinterpret_cast<float2*>(to + lines * D + 2 * all) = make_float2(m, ok ? l : NAN);
                if (tid == 0) to[lines * (D + 2)] = sm.bad_values ? 1.0f : 0.0f;
            } else if (NQ == 2) {
                // the only sums of a row that this CTA has: they go to the CTA that writes the row, a thread a row
                const int row = g * ROWS + r, i = share_of(row), owner = row - i * parts;
                const unsigned to = ib_cluster_address(inbox + (part * most + i) * Sh::OLD, owner);
#pragma unroll 1
                for (int e = 0; e < D; e += 32) {
                    unsigned x[32];
                    __syncwarp();
                    tmem_ld32(o_at + e, x);
                    if (!mine) continue;
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        remote_store(to + (e + k) * 4, make_float4(__uint_as_float(x[k]), __uint_as_float(x[k + 1]), __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3])));
                }
                if (mine) remote_store(ib_cluster_address(inbox_ml + (part * most + i) * 4, owner), make_float4(m, ok ? l : NAN, sm.bad_values ? 1.0f : 0.0f, 0.0f));
            } else {
                if (count > 0 && ok) {
                    float* row = sums + (g * ROWS + r) * Sh::OLD;
#pragma unroll
                    for (int e = 0; e < D; e += 32) {
                        unsigned x[32];
                        tmem_ld32(o_at + e, x);
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<uint4*>(row + e + k) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                    }
                }
                part_m[g * ROWS + r] = m;
                part_l[g * ROWS + r] = ok ? l : NAN;
            }
        } else if (scratch == nullptr && parts > 1) {
            ib_cluster_sync();
        }
        fence_before();
    }
    if (warp >= PRODUCERS && scratch == nullptr && parts > 1) ib_cluster_sync();
    __syncthreads();
    if (warp == ISSUER) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    if ((scratch != nullptr && parts > 1) || (NQ == 2 && parts == 1 && !sm.bad_values)) return;
    // Join: first the sums that this CTA has of a row (of two streams), which go to the CTA that writes the row (every parts-th),
    // and there those of the cluster's CTAs.  What goes out is not waited for; a look into another CTA's memory takes 700 cycles.  Eight lanes
    // a row, and loops as they stand: this code runs once, and unrolled ones wait for their instructions (ten cycles each) longer than they
    // save.  Every sum comes in the same order whatever the grid.
    constexpr int QUADS = D / 32, PASS = THREADS / 8;
    const int line0 = tid >> 3, e = (lane & 7) * 4;              // a lane's numbers: e .. e + 3 and every 32 behind them
    if (NQ == 1) {
#pragma unroll 1
        for (int row = line0; row < rows; row += PASS) {
            float4 o[QUADS] = {};
            float top = -INFINITY, total = 0.0f;
#pragma unroll 1
            for (int line = row; line < 2 * ROWS; line += ROWS)
                join<QUADS>(top, total, o, part_m[line], part_l[line], sums + line * Sh::OLD + e);
            const int i = share_of(row), owner = row - i * parts;
            const unsigned to = ib_cluster_address(inbox + (part * most + i) * Sh::OLD + e, owner);
#pragma unroll
            for (int k = 0; k < QUADS; ++k) remote_store(to + k * 128, o[k]);
            if (e == 0) remote_store(ib_cluster_address(inbox_ml + (part * most + i) * 4, owner), make_float4(top, total, sm.bad_values ? 1.0f : 0.0f, 0.0f));
        }
    }
    if (parts > 1) ib_cluster_sync();
    else __syncthreads();
#pragma unroll 1
    for (int i = line0; part + i * parts < rows; i += PASS) {
        float4 o[QUADS] = {};
        float top = -INFINITY, total = 0.0f, bad = 0.0f;
#pragma unroll 1
        for (int p = 0; p < parts; ++p) {
            const int at = p * most + i;
            const float4 ml = *reinterpret_cast<const float4*>(inbox_ml + at * 4);
            bad = fmaxf(bad, ml.z);
            join<QUADS>(top, total, o, ml.x, ml.y, inbox + at * Sh::OLD + e);
        }
        write_row<D, QUADS>(A, S, place, first_row + part + i * parts, head, e, 32, o, total, bad != 0.0f, t_first, all_tiles, lo_max);
    }
}

// The rows whose keys were cut into slices by CTAs that do not run together: their sums lie in memory, slice by slice.  A thread
// takes 16 numbers of a row, a warp 32 rows.
template <int D, int NQ>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ Args A, int slices, int slice_rows, const float* __restrict__ scratch) {
    constexpr int CHUNKS = NQ * ROWS * (D / 16) / 256, STREAMS = NQ == 1 ? 2 : 1;      // that have a row's sums
    const int unit = blockIdx.x / CHUNKS, at = blockIdx.x % CHUNKS * 256 + threadIdx.x, row = at % (NQ * ROWS), e = at / (NQ * ROWS) * 16;
    const int head = unit % A.n_kv, row_tile = unit / A.n_kv % A.tiles_of_rows, req = unit / A.n_kv / A.tiles_of_rows;
    const Span S = span_of(A, req);
    const int group = A.group, first_row = row_tile * (NQ * ROWS);
    const int rows = min(S.n_tree * group - first_row, slice_rows), lines = Shape<D, NQ>::lines(slice_rows), sums = Shape<D, NQ>::slice_sums(slice_rows);
    if (row >= rows) return;
    int lo_min = 0, lo_max = 0;
    if (A.span != 0) {
        lo_min = 0x7fffffff;
#pragma unroll 1
        for (int t = first_row / group; t <= (first_row + rows - 1) / group; ++t) {
            const int lo = first_key(A, S, t);
            lo_min = min(lo_min, lo);
            lo_max = max(lo_max, lo);
        }
        lo_min = min(lo_min, S.context);
    }
    const int t_first = lo_min / KEYS, all_tiles = (S.keys + KEYS - 1) / KEYS - t_first, parts = slices_of(all_tiles, slices);
    if (parts == 1) return;           // (its rows are written)
    float4 o[4] = {};
    float top = -INFINITY, total = 0.0f;
    bool bad_values = false;
    const float* from = scratch + (long)unit * slices * sums;
#pragma unroll 2
    for (int p = 0; p < parts * STREAMS; ++p) {
        const float* slice = from + (long)(p / STREAMS) * sums;
        const int line = row + p % STREAMS * slice_rows;
        const float2 ml = *reinterpret_cast<const float2*>(slice + lines * D + 2 * line);
        bad_values |= slice[lines * (D + 2)] != 0.0f;
        join<4>(top, total, o, ml.x, ml.y, slice + (e / 4 * lines + line) * 4, lines * 4);
    }
    const Place place = {A.table + (long)req * A.max_pages, head, S.keys};
    write_row<D, 4>(A, S, place, first_row + row, head, e, 4, o, total, bad_values, t_first, all_tiles, lo_max);
}

// How a call is cut: row tiles of NQ x 128 rows, a part of the keys for each CTA, in clusters or (waves) in slices
struct Cut { long pairs, parts; int tiles_of_rows, tiles, slice_rows; bool waves; };

template <int D, int NQ>
static int cut_of(const Args& A, int max_tree, int max_keys, Cut& c) {
    static IbDeviceSet done;
    if (const int code = ib_allow_dynamic_smem(done, tree_kernel<D, NQ>, Shape<D, NQ>::SMEM)) return code;
    c.tiles_of_rows = (int)(((long)max_tree * (A.n_heads / A.n_kv) + NQ * ROWS - 1) / (NQ * ROWS));
    c.pairs = (long)A.n_requests * A.n_kv * c.tiles_of_rows;
    long keys = max_keys;
    if (A.span > 0 && keys > (long)A.span + max_tree + KEYS) keys = (long)A.span + max_tree + KEYS;
    c.tiles = (int)((keys + KEYS - 1) / KEYS);
    // One wave of CTAs: as many parts as there are SMs for, a cluster each.  More than that: requests differ in length, and clusters would wait
    // for as many free SMs at once; slices of 24 tiles or more, the longest requests first, are joined by a kernel of their own.  (Trees of 64,
    // 32 heads on 8, 16 requests of 100 to 16,384 keys: slices of 12, 16, 24, 32 tiles 190, 180, 167, 178 us in short runs, whole requests 246; all of 16,384:
    // 325, 306, 305, 299; of 100 to 4,500: 67, 73, and whole ones, which 24 leaves them, 73.)
    c.waves = 2 * c.pairs > 148 && c.tiles > 2 * SLICE;
    c.parts = c.waves ? (c.tiles + SLICE - 1) / SLICE : 148 / c.pairs;
    if (c.parts > c.tiles) c.parts = c.tiles;
    // A slice has lines for the rows that a tile of the largest tree has, 32 by 32 as warps write them, and all slices together have 256 MB: the longest
    // request may be one of many short ones, for which as many slices are set aside, and CTAs that find none cost time too.  (No bound, 1 GB, 256,
    // 64 MB: 64 requests of up to 2,000 keys and one of 131,072, trees of 4, 699 MB without: 554, 554, 298, 547 us; trees of 40, 1,748 MB: 564, 410, 314,
    // 1,782; 256 requests, trees of 4, 2,796 MB: 3,216, 1,358, 554, 1,700; 100 requests of 100 to 32,400 keys, trees of 40: 1,647, 1,645, 1,538, 1,412.)
    const long rows = (long)max_tree * (A.n_heads / A.n_kv);
    c.slice_rows = c.waves && rows < NQ * ROWS ? (int)(rows + 31) / 32 * 32 : NQ * ROWS;
    long most = IB_MAX_CLUSTER;
    if (c.waves) {
        most = MOST_SCRATCH / (c.pairs * Shape<D, NQ>::slice_sums(c.slice_rows) * 4L);
        if (most > MOST_SLICES) most = MOST_SLICES;
        if (most < 2) {               // (whole requests)
            c.waves = false;
            c.slice_rows = NQ * ROWS;
            most = 1;
        }
    }
    c.parts = c.parts < 1 ? 1 : c.parts > most ? most : c.parts;
    // (Clusters that do not all run at once take twice the time: 5 requests of 20 pairs with a window 26.2 us in clusters of seven, 16.2 in six.)
    static IbClusters clusters;
    while (!c.waves && c.parts > 1 && ib_clusters_at_once(clusters, tree_kernel<D, NQ>, (int)c.parts, THREADS, Shape<D, NQ>::SMEM) < c.pairs) --c.parts;
    return IB_OK;
}

template <int D, int NQ>
static long launch(Args A, const Cut& c, void* workspace, bool ask, cudaStream_t stream) {
    const long pairs = c.pairs, parts = c.parts;
    A.tiles_of_rows = c.tiles_of_rows;
    const long needed = c.waves ? pairs * parts * Shape<D, NQ>::slice_sums(c.slice_rows) * 4 : 0;
    if (ask) return needed;
    float* scratch = needed ? static_cast<float*>(workspace) : nullptr;
    if (needed && workspace == nullptr) return IB_ERR_ARGUMENT;
    // boxes of a page's places, or of 128 in larger pages, where whole ones make a tile and start on eight rows
    int box = A.page_shift >= 3 ? (A.page_size < KEYS ? A.page_size : KEYS) : 0;
    CUtensorMap map_k = {}, map_v = {};
    if (box > 0) {
        const EncodeTiled encode = encode_fn();
        const cuuint64_t dims[2] = {D, (cuuint64_t)A.n_pages * A.n_kv * A.page_size}, strides[1] = {D * 2};
        const cuuint32_t sizes[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
        for (int values = 0; values < 2 && box > 0; ++values)
            if (dims[1] == 0 || encode == nullptr
                || encode(values ? &map_v : &map_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(values ? A.v : A.k), dims, strides, sizes, steps,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                       != CUDA_SUCCESS)
                box = 0;
    }
    const int ranked = A.n_requests > 1 && A.n_requests <= RANKED && pairs * parts > 148;
    const int code = launch_cluster(tree_kernel<D, NQ>, pairs * parts, scratch ? 1 : (int)parts, THREADS, Shape<D, NQ>::SMEM, stream, map_k, map_v, A,
                                    (int)parts, ranked, box, scratch, c.slice_rows);
    if (code != IB_OK || scratch == nullptr) return code;
    const long blocks = pairs * (NQ * ROWS * (D / 16) / 256);
    if (blocks > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    tree_join_kernel<D, NQ><<<(unsigned)blocks, 256, 0, stream>>>(A, (int)parts, c.slice_rows, scratch);
    return ib_launch_status();
}

// Two sets of rows share a CTA's keys, or each has CTAs of its own, with half as many parts and a shorter start and join.  In tiles of keys a CTA,
// n1 and n2, one set takes about 10 + 1.25 n1 us and two take 14 + 1.85 n2.  (Trees of 64, 32 heads on 8 of 128; one set and two: 1 request of 2,000
// keys 15.0 and 21.5 us, 4 21.5 and 23.7, 8 31.6 and 28.9; 4 of 30,000 156 and 117.  5 chains of 37, 20 heads on 4 of 64, window 1,500: 15.0 and 16.2.)
template <int D>
static long launch(const Args& A, int max_tree, int max_keys, void* workspace, bool ask, cudaStream_t stream) {
    Cut one, two;
    if (const int code = cut_of<D, 1>(A, max_tree, max_keys, one)) return code;
    if ((long)max_tree * (A.n_heads / A.n_kv) > ROWS) {
        if (const int code = cut_of<D, 2>(A, max_tree, max_keys, two)) return code;
        const long n1 = one.waves ? one.pairs * one.tiles / 148 : (one.tiles + one.parts - 1) / one.parts, n2 = (two.tiles + two.parts - 1) / two.parts;
        if (2 * two.pairs > 148 || 2 * n1 > 3 * n2 + 6) return launch<D, 2>(A, two, workspace, ask, stream);
    }
    return launch<D, 1>(A, one, workspace, ask, stream);
}

}  // namespace tree_tc

long ib_tree_tcgen05(tree::Args A, int max_tree, int max_keys, void* workspace, bool ask, cudaStream_t stream) {
    using namespace tree_tc;
    const uintptr_t at = reinterpret_cast<uintptr_t>(A.q) | reinterpret_cast<uintptr_t>(A.k) | reinterpret_cast<uintptr_t>(A.v);
    if ((A.dim != 64 && A.dim != 128) || at % 16 || !(A.scale_log2 > 0.0f)) return IB_ERR_UNSUPPORTED;
    return A.dim == 128 ? launch<128>(A, max_tree, max_keys, workspace, ask, stream) : launch<64>(A, max_tree, max_keys, workspace, ask, stream);
}

IB_EXPORT int ib_attention_tree_error(int reset) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, tree_tc::g_error, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(tree_tc::g_error, &zero, sizeof(int));
    }
    return v;
}
IB_EXPORT int ib_attention_tree_error_async(int* out, cudaStream_t stream) {
    return (int)cudaMemcpyFromSymbolAsync(out, tree_tc::g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}
