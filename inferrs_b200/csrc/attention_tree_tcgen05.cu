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
// What bounds it is what comes from memory: a tile of 128 keys and values of 128 numbers is 64 KB, 2,900 cycles of an SM's share of the
// copy bandwidth, and needs 1,100 cycles of products and as many of exponentials for every 128 rows.  Keys and values come through
// a ring of tiles that four warps fill with cp.async, 16 bytes a lane: rows of a page lie anywhere, pages have any size, and where there is
// no key zeros are written.  Ring places come in the order in which the products take them.
//
// What no row sees must not reach it: a product cannot leave a value out, and 0 times infinity is no number.  So in tiles that some row does
// not see in full the warps that fill the ring look at the values that they brought, put zeros in the place of those that are
// infinite or no numbers, and the rows that see such a value get it added at the end, from its page.
#include "sm100.cuh"
#include "tree.cuh"

namespace tree_tc {

using namespace sm100;
using namespace tree;
typedef __nv_bfloat16 bf16;

constexpr int ROWS = 128, KEYS = 128;
constexpr int PRODUCERS = 8, ISSUER = 12, THREADS = 13 * 32;      // warps 0..7: softmax, 8..11: the ring, 12: products
constexpr float STEP = 8.0f;          // how far (log2) a row's maximum may outgrow its reference
constexpr int MOST_PARTS = 8;
constexpr int RANKED = 1024;          // requests that are put in order of their length

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
    static constexpr int SMEM = 1024 + TILES + 256;
    static_assert(SUMS + 4 * ROWS * 4 <= TILES, "the sums, references and denominators take the place of the tiles");
    // one CTA an SM: a second one would wait for the first one's tensor memory while others of its cluster wait for it
    static_assert(SMEM > 116 * 1024 && SMEM <= 232448, "one CTA an SM");
};

struct Small {                 // what stands behind the tiles
    unsigned long long full[8], empty[8], s_full[2], p_full[2], o_full, q_full;
    unsigned tmem;
    int req, lo_min, lo_max, bad_values;
};
static_assert(sizeof(Small) <= 256, "");

__device__ __forceinline__ void cp16(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// an arrival when all that this thread has asked for so far is there
__device__ __forceinline__ void cp_arrive(unsigned bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Vectors of D numbers to rows 32 w .. 32 w + 31 of a tile; `index` is the place of this lane's row among the vectors at `base` (-1: zeros)
template <int D>
__device__ __forceinline__ void load_rows(unsigned tile, const bf16* base, int index, int w, int lane) {
    constexpr int CHUNKS = D / 8, STEP_ROWS = 32 / CHUNKS;
    const int c = lane % CHUNKS, sub = lane / CHUNKS;
    const unsigned at = tile + (unsigned)((c >> 3) * (ROWS * 128) + w * 32 * 128);
#pragma unroll
    for (int i = 0; i < 32 / STEP_ROWS; ++i) {
        const int r = i * STEP_ROWS + sub;
        const int from = __shfl_sync(0xffffffffu, index, r);
        cp16(at + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (long)(from < 0 ? 0 : from) * D + c * 8, from < 0 ? 0 : 16);
    }
}

// Zeros for what is no finite number among what this lane has loaded with load_rows; true if there was any
template <int D>
__device__ __forceinline__ bool clean_rows(unsigned tile, int w, int lane) {
    constexpr int CHUNKS = D / 8, STEP_ROWS = 32 / CHUNKS;
    const int c = lane % CHUNKS, sub = lane / CHUNKS;
    const unsigned at = tile + (unsigned)((c >> 3) * (ROWS * 128) + w * 32 * 128);
    bool any = false;
#pragma unroll 4
    for (int i = 0; i < 32 / STEP_ROWS; ++i) {
        const int r = i * STEP_ROWS + sub;
        const unsigned a = at + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        unsigned v[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
        unsigned hit = 0;      // bit 15 of a half carries over where all bits of its exponent are set
#pragma unroll
        for (int k = 0; k < 4; ++k) hit |= ((v[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        if (hit) {
            any = true;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned h = ((v[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                v[k] &= ~((h >> 15) * 0xffffu);
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
        }
    }
    return any;
}

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

// which of the 32 keys from jb on a row sees; lo: the first key of the context that it sees
__device__ unsigned visible(const Args& A, const Span& S, const Place& p, const int* words, int lo, int jb, bool bad_pages) {
    const int a = max(lo - jb, 0), b = min(S.context - jb, 32);
    unsigned bits = 0;
    if (b > a) bits = (b == 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u);
    if (jb + 32 > S.context) {
        unsigned drafted = mask_bits(A, S, words, jb - S.context);
        const int left = S.keys - jb;
        if (left < 32) drafted &= left <= 0 ? 0u : (1u << left) - 1u;
        bits |= drafted;
    }
    if (bad_pages)
        for (int k = 0; k < 32; ++k)
            if ((bits >> k & 1u) && key_index(A, p, jb + k) < 0) bits &= ~(1u << k);
    return bits;
}

__device__ __forceinline__ float4 remote_f32x4(const float* local, unsigned rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float2 remote_f32x2(const float* local, unsigned rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote(local, rank)) : "memory");
    return v;
}

template <int D, int NQ>
__global__ void __launch_bounds__(THREADS, 1) tree_kernel(const Args A, int parts, int ranked) {
    typedef Shape<D, NQ> Sh;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    float* sums = reinterpret_cast<float*>(smem);                 // [2][ROWS][OLD], once the tiles have been used
    float* part_m = reinterpret_cast<float*>(smem + Sh::SUMS);    // [2][ROWS]
    float* part_l = part_m + 2 * ROWS;
    Small& sm = *reinterpret_cast<Small*>(smem + Sh::TILES);
    const unsigned sq = smem_u32(smem), ring = sq + NQ * Sh::TILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    int unit = blockIdx.x / parts;
    const int part = blockIdx.x - unit * parts;
    const int head = unit % A.n_kv;
    unit /= A.n_kv;
    const int row_tile = unit % A.tiles_of_rows;
    int req = unit / A.tiles_of_rows;
    if (ranked) {                     // the longest contexts first: the grid's last CTAs are short ones
        int* lengths = reinterpret_cast<int*>(smem);
        for (int i = tid; i < A.n_requests; i += THREADS) lengths[i] = A.context[i];
        __syncthreads();
        for (int i = tid; i < A.n_requests; i += THREADS) {
            const int mine = lengths[i];
            int ahead = 0;
            for (int j = 0; j < A.n_requests; ++j) ahead += lengths[j] > mine || (lengths[j] == mine && j < i);
            if (ahead == req) sm.req = i;
        }
        __syncthreads();
        req = sm.req;
    }
    const Span S = span_of(A, req);
    const int group = A.n_heads / A.n_kv;
    const int first_row = row_tile * (NQ * ROWS);
    const int rows = min(S.n_tree * group - first_row, NQ * ROWS);
    if (rows <= 0) return;            // (the whole cluster leaves)

    if (tid == 0) {
        sm.lo_min = 0x7fffffff;
        sm.lo_max = 0;
        sm.bad_values = 0;
    }
    if (warp == ISSUER) {
        if (lane == 0) {
            for (int i = 0; i < Sh::STAGES; ++i) { mbar_init(smem_u32(&sm.full[i]), 128); mbar_init(smem_u32(&sm.empty[i]), 1); }
            for (int g = 0; g < 2; ++g) {
                const int used = NQ == 2 ? rows - g * ROWS : rows;
                mbar_init(smem_u32(&sm.s_full[g]), 1);
                mbar_init(smem_u32(&sm.p_full[g]), used <= 0 ? 1 : used >= ROWS ? 4 : (used + 31) / 32);
            }
            mbar_init(smem_u32(&sm.o_full), 1);
            mbar_init(smem_u32(&sm.q_full), 128);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (A.span != 0) {                // the first keys that the CTA's rows see: the least and the greatest
        const int t0 = first_row / group, t1 = (first_row + rows - 1) / group;
        for (int t = t0 + tid; t <= t1; t += THREADS) {
            const int lo = first_key(A, S, t);
            atomicMin(&sm.lo_min, lo);
            atomicMax(&sm.lo_max, lo);
        }
        __syncthreads();
    }
    const int lo_min = A.span != 0 ? min(sm.lo_min, S.context) : 0, lo_max = A.span != 0 ? sm.lo_max : 0;
    const unsigned tmem = sm.tmem;
    const int t_first = lo_min / KEYS, all_tiles = (S.keys + KEYS - 1) / KEYS - t_first;
    const int t_begin = t_first + (int)((long)all_tiles * part / parts), t_end = t_first + (int)((long)all_tiles * (part + 1) / parts);
    const int n = t_end - t_begin;
    // tiles that each stream takes
    const int count0 = NQ == 2 ? n : (n + 1) / 2, count1 = NQ == 2 ? (rows > ROWS ? n : 0) : n / 2;
    const Place place = {A.table + (long)req * A.max_pages, head, S.keys};
    // keys that some row does not see
    auto partly = [&](int t) { return t * KEYS < lo_max || (t + 1) * KEYS > S.context; };
    bool ok = true;

    if (warp >= PRODUCERS && warp < ISSUER) {
        const int w = warp - PRODUCERS;
        const bf16* q = static_cast<const bf16*>(A.q);
#pragma unroll
        for (int g = 0; g < NQ; ++g) {
            const int r = g * ROWS + w * 32 + lane;
            int index = -1;
            if (r < rows) {
                const int at = first_row + r, token = at / group;
                index = (S.row0 + token) * A.n_heads + head * group + at - token * group;
            }
            load_rows<D>(sq + g * Sh::TILE, q, index, w, lane);
        }
        cp_arrive(smem_u32(&sm.q_full));
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
        bool values = false;
        int t = 0, index = -1;
        if (n > 0) {
            t = tile_of(0, values);
            index = key_index(A, place, (t_begin + t) * KEYS + w * 32 + lane);
        }
        int slot = 0, turn = 0;
        for (int e = 0; e < 2 * n; ++e) {
            if (turn > 0 && !mbar_wait(smem_u32(&sm.empty[slot]), (turn - 1) & 1, 1)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const unsigned dst = ring + slot * Sh::TILE, bar = smem_u32(&sm.full[slot]);
            load_rows<D>(dst, static_cast<const bf16*>(values ? A.v : A.k), index, w, lane);
            if (values && partly(t_begin + t)) {
                cp_wait_all();
                if (clean_rows<D>(dst, w, lane)) sm.bad_values = 1;
                mbar_arrive(bar);
            } else {
                cp_arrive(bar);
            }
            if (e + 1 < 2 * n) {
                t = tile_of(e + 1, values);
                index = key_index(A, place, (t_begin + t) * KEYS + w * 32 + lane);
            }
            if (++slot == Sh::STAGES) { slot = 0; ++turn; }
        }
        cp_wait_all();
    } else if (warp == ISSUER) {
        if (lane == 0) {
            constexpr unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(ROWS >> 4) << 24);
            constexpr unsigned idesc_s = idesc | ((unsigned)(KEYS >> 3) << 17), idesc_o = idesc | (1u << 16) | ((unsigned)(D >> 3) << 17);
            auto k_entry = [&](int t) { return NQ == 2 ? 2 * t : t == 0 ? 0 : 2 * t - 1; };
            auto v_entry = [&](int t) { return NQ == 2 ? 2 * t + 1 : min(2 * t + 2, 2 * n - 1); };
            const int last = NQ == 2 && count1 > 0 ? 1 : 0;            // with two sets of rows: the stream that is done with a tile last
            auto arrived = [&](int e) {
                if (!mbar_wait(smem_u32(&sm.full[e % Sh::STAGES]), (e / Sh::STAGES) & 1, 2)) return false;
                fence_async();
                fence_after();
                return true;
            };
            auto scores = [&](int g, int i) {                          // of the stream's i-th tile
                const int e = k_entry(NQ == 2 ? i : 2 * i + g);
                if (!arrived(e)) return false;
                const unsigned k = ring + (e % Sh::STAGES) * Sh::TILE, rows_q = sq + (NQ == 2 ? g * Sh::TILE : 0);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    const unsigned off = (s >> 2) * (ROWS * 128) + (s & 3) * 32;
                    umma(tmem + g * 128, desc_k_major(rows_q + off), desc_k_major(k + off), idesc_s, s != 0);
                }
                umma_commit(smem_u32(&sm.s_full[g]));
                if (NQ == 1 || g == last) umma_commit(smem_u32(&sm.empty[e % Sh::STAGES]));
                return true;
            };
            ok = mbar_wait(smem_u32(&sm.q_full), 0, 3);
            for (int g = 0; g < 2 && ok; ++g)
                if ((g ? count1 : count0) > 0) ok = scores(g, 0);
            for (int i = 0; i < count0 && ok; ++i) {
                for (int g = 0; g < 2 && ok; ++g) {
                    if (i >= (g ? count1 : count0)) continue;
                    const int e = v_entry(NQ == 2 ? i : 2 * i + g);
                    if (!mbar_wait(smem_u32(&sm.p_full[g]), i & 1, 4) || !arrived(e)) { ok = false; break; }
                    const unsigned v = ring + (e % Sh::STAGES) * Sh::TILE;
#pragma unroll
                    for (int s = 0; s < KEYS / 16; ++s)
                        umma_ts(tmem + 256 + g * 128, tmem + g * 128 + s * 8, desc_mn_major(v + s * 16 * 128, ROWS * 128), idesc_o, (i | s) != 0);
                    if (NQ == 1 || g == last) umma_commit(smem_u32(&sm.empty[e % Sh::STAGES]));
                    if (i + 1 < (g ? count1 : count0)) ok = scores(g, i + 1);
                }
            }
            umma_commit(smem_u32(&sm.o_full));
        }
        __syncwarp();
    } else {
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
                for (int slot = j0 / A.page_size + lane; (long)slot * A.page_size < j1; slot += 32) {
                    const int page = place.bt[slot];
                    if (page < 0 || page >= A.n_pages) bad = true;
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
            const unsigned s_at = tmem + lanes + g * 128, o_at = tmem + lanes + 256 + g * 128;
            float m = -INFINITY, l = 0.0f;
            for (int i = 0; i < count; ++i) {
                if (!mbar_wait(smem_u32(&sm.s_full[g]), i & 1, 5)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                const int t = t_begin + (NQ == 2 ? i : 2 * i + g), j0 = t * KEYS;
                const bool plain = __all_sync(0xffffffffu, !bad && j0 >= lo && j0 + KEYS <= S.context);
                unsigned see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                if (!plain) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) see[c] = visible(A, S, place, words, lo, j0 + 32 * c, bad);
                }
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    unsigned x[32];
                    tmem_ld32_issue(s_at + 32 * c, x);
                    tmem_ld_wait();
                    if (!plain) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(see[c] >> k & 1u)) x[k] = 0xff800000u;
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) top4[k & 3] = fmaxf(top4[k & 3], __uint_as_float(x[k]));
                }
                const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * A.scale_log2;     // (the scale is positive)
                const bool move = top > m + STEP || (m == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float c = move ? (m == -INFINITY ? 0.0f : ex2(m - top)) : 1.0f;
                    if (i > 0) {      // (the stream's products are done: the one that gave S came behind them)
#pragma unroll 1
                        for (int e = 0; e < D; e += 32) {
                            unsigned x[32];
                            tmem_ld32_issue(o_at + e, x);
                            tmem_ld_wait();
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
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    unsigned x[32], p[16];
                    tmem_ld32_issue(s_at + 32 * c, x);
                    tmem_ld_wait();
                    if (!plain) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(see[c] >> k & 1u)) x[k] = 0xff800000u;
                    }
                    float add[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float a = ex2(fmaf(__uint_as_float(x[2 * k]), A.scale_log2, -ref));
                        const float b = ex2(fmaf(__uint_as_float(x[2 * k + 1]), A.scale_log2, -ref));
                        add[0] += a;
                        add[1] += b;
                        p[k] = pack_bf16(a, b);
                    }
                    l += add[0] + add[1];
                    tmem_st16(s_at + 16 * c, p);
                }
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[g]));
            }
            if (!mbar_wait(smem_u32(&sm.o_full), 0, 6)) ok = false;       // every product is done: the tiles' memory is free
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            if (count > 0 && ok) {
                float* row = sums + (g * ROWS + r) * Sh::OLD;
#pragma unroll
                for (int e = 0; e < D; e += 32) {
                    unsigned x[32];
                    tmem_ld32_issue(o_at + e, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<uint4*>(row + e + k) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                }
            }
            part_m[g * ROWS + r] = m;
            part_l[g * ROWS + r] = l;
        }
        fence_before();
    }
    cluster_sync();
    if (warp == ISSUER) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    // join: CTA `part` writes every parts-th row; a lane holds D / 32 neighbouring numbers of a row
    constexpr int PER = D / 32, STREAMS = NQ == 2 ? 1 : 2;
    bool bad_values = false;
    for (int c = 0; c < parts; ++c) {
        int v;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote(&sm.bad_values, c)) : "memory");
        bad_values |= v != 0;
    }
    for (int row = part + warp * parts; row < rows; row += parts * (THREADS / 32)) {
        const int g0 = NQ == 2 ? row / ROWS : 0, r = row - g0 * ROWS;
        // lane p looks at the p-th of the row's sums
        const int n_sums = parts * STREAMS;
        float m = -INFINITY, l = 0.0f;
        if (lane < n_sums) {
            m = remote_f32(&part_m[(g0 + lane % STREAMS) * ROWS + r], lane / STREAMS);
            l = remote_f32(&part_l[(g0 + lane % STREAMS) * ROWS + r], lane / STREAMS);
        }
        const float top = ib_warp_max(m), ref = top == -INFINITY ? 0.0f : top;
        const float f = l == 0.0f ? 0.0f : ex2(m - ref);
        const float total = ib_warp_sum(l == 0.0f ? 0.0f : l * f);
        float o[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = 0.0f;
        for (int p = 0; p < n_sums; ++p) {
            if (__shfl_sync(0xffffffffu, l, p) == 0.0f) continue;         // none of its keys is seen
            const float fp = __shfl_sync(0xffffffffu, f, p);
            const float* from = sums + ((g0 + p % STREAMS) * ROWS + r) * Sh::OLD + lane * PER;
            if constexpr (PER == 4) {
                const float4 x = remote_f32x4(from, p / STREAMS);
                o[0] = fmaf(x.x, fp, o[0]); o[1] = fmaf(x.y, fp, o[1]); o[2] = fmaf(x.z, fp, o[2]); o[3] = fmaf(x.w, fp, o[3]);
            } else {
                const float2 x = remote_f32x2(from, p / STREAMS);
                o[0] = fmaf(x.x, fp, o[0]); o[1] = fmaf(x.y, fp, o[1]);
            }
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] *= inv;
        const int at = first_row + row, token = at / group;
        if (bad_values) {             // infinite values and no numbers that the row sees in tiles that not all rows see
            const int lo = first_key(A, S, token);
            const int* words = A.seen + (long)(S.row0 + token) * A.words;
            for (int t = t_first; t < t_first + all_tiles; ++t) {
                if (!partly(t)) continue;
                for (int c = 0; c < 4; ++c) {
                    unsigned see = visible(A, S, place, words, lo, t * KEYS + 32 * c, true);
                    for (; see; see &= see - 1) {
                        const int index = key_index(A, place, t * KEYS + 32 * c + __ffs(see) - 1);
#pragma unroll
                        for (int e = 0; e < PER; ++e) {
                            const float v = __bfloat162float(static_cast<const bf16*>(A.v)[(long)index * D + lane * PER + e]);
                            if (!(fabsf(v) < INFINITY)) o[e] += v;
                        }
                    }
                }
            }
        }
        bf16* dst = static_cast<bf16*>(A.out) + (long)(S.row0 + token) * A.out_ld + (long)(head * group + at - token * group) * D + lane * PER;
        unsigned packed[PER / 2];
#pragma unroll
        for (int e = 0; e < PER; e += 2) packed[e / 2] = pack_bf16(o[e], o[e + 1]);
        if ((reinterpret_cast<uintptr_t>(A.out) | (uintptr_t)(A.out_ld * 2)) % (PER * 2) == 0) {
            if constexpr (PER == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
            else *reinterpret_cast<unsigned*>(dst) = packed[0];
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) dst[e] = __float2bfloat16_rn(o[e]);
        }
    }
    cluster_sync();                   // nobody leaves while others read its sums
}

template <int D, int NQ>
static int launch(Args A, int max_tree, int max_keys, cudaStream_t stream) {
    static IbDeviceSet done;
    if (const int code = ib_allow_dynamic_smem(done, tree_kernel<D, NQ>, Shape<D, NQ>::SMEM)) return code;
    A.tiles_of_rows = (int)(((long)max_tree * (A.n_heads / A.n_kv) + NQ * ROWS - 1) / (NQ * ROWS));
    const long pairs = (long)A.n_requests * A.n_kv * A.tiles_of_rows;
    const int tiles = (max_keys + KEYS - 1) / KEYS;
    long parts = 148 / pairs;
    if (parts > tiles) parts = tiles;
    parts = parts < 1 ? 1 : parts > MOST_PARTS ? MOST_PARTS : parts;
    const int ranked = A.n_requests > 1 && A.n_requests <= RANKED && pairs * parts > 148;
    return launch_cluster(tree_kernel<D, NQ>, pairs * parts, (int)parts, THREADS, Shape<D, NQ>::SMEM, stream, A, (int)parts, ranked);
}

}  // namespace tree_tc

int ib_tree_tcgen05(tree::Args A, int max_tree, int max_keys, cudaStream_t stream) {
    using namespace tree_tc;
    const uintptr_t at = reinterpret_cast<uintptr_t>(A.q) | reinterpret_cast<uintptr_t>(A.k) | reinterpret_cast<uintptr_t>(A.v);
    if ((A.dim != 64 && A.dim != 128) || at % 16 || !(A.scale_log2 > 0.0f)) return IB_ERR_UNSUPPORTED;
    const bool two = (long)max_tree * (A.n_heads / A.n_kv) > ROWS;
    if (A.dim == 128) return two ? launch<128, 2>(A, max_tree, max_keys, stream) : launch<128, 1>(A, max_tree, max_keys, stream);
    return two ? launch<64, 2>(A, max_tree, max_keys, stream) : launch<64, 1>(A, max_tree, max_keys, stream);
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
