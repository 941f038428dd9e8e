// Log probabilities of given tokens, the distribution's entropy and its most likely tokens, for every row of logits.
//
// With m the row's largest logit, z = x - m, S = sum e^z and W = sum e^z z (kept in powers of two):
//   log p(t) = z_t - log S        entropy = -sum p log p = log S - W / S
// S and W are sums of numbers of one sign and lose nothing to cancellation.  Every thread keeps m, S and W of what it has seen
// in 32 bits; when its m grows by g, S becomes S e^-g and W becomes (W - S g) e^-g.  A logit that is no number counts as minus
// infinity, as it does for the sampler; a row whose largest logit is infinite has no distribution, and NaN as its numbers.
//
// The logits are read once.  The k most likely tokens come out of the same pass, by blocks of 16 neighbouring logits, a thread's share of a
// chunk: the k blocks whose largest logits are the largest (of equal ones the earlier block) hold the k most likely tokens, because every block
// ahead of a token's own has a token that is ahead of it.  A block's key is its largest logit's bits made ascending, the complement of its place
// below them.  A bound that at least k keys reach is kept; the key of a block that passes it is noted in shared memory, and behind chunks
// 2, 5, 11 .. the k best of the noted ones give a higher bound.  The first bound is the k-th largest of 64 groups' largest keys; expected are k
// to 2 k notes from the first 4,096 logits and k more for every doubling behind them.  At the end the k blocks are looked through.
//
// Many rows of 32 bits are bound by memory: 2,048 rows of 151,936 logits take 179 us without and 191 with the most likely token (190 at the
// copy rate, which counts a write for every read), 218 with the 32 most likely ones; in bfloat16, which are half the bytes, the instructions
// bound it (172 us with five).  A warp of its own fetches (bulk copies into 64 KB, three CTAs an SM), and a logit costs one exponential and half
// of a packed instruction of each other kind.  Few rows are bound by the chain from the first copy through the bounds to the join of a row's CTAs:
// one row takes 6.6 us, 10 with the five most likely tokens.
#include "clusters.cuh"
#include "sm100.cuh"

namespace lp {

constexpr int THREADS = 256;         // that look at logits; one warp more fetches them
constexpr int RING = 4096;           // 16-byte vectors that may be on their way or waiting
constexpr int MAX_TOP = 32;
constexpr int NOTES = 1024;          // room for noted keys
constexpr int GROUPS = 64;           // groups of 4 threads whose largest keys give the first bound
constexpr float LOWEST = -300.0f;    // 2^-300 is 0 in 32 bits, and 0 times it is 0

typedef unsigned long long u64;

__device__ __forceinline__ u64 key_of(float x, int at) {
    const unsigned b = __float_as_uint(x + 0.0f);      // (of two zeros none is the larger one)
    const unsigned up = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((u64)up << 32) | (unsigned)~at;
}
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned up = (unsigned)(key >> 32);
    return __uint_as_float((up & 0x80000000u) ? (up & 0x7fffffffu) : ~up);
}
__device__ __forceinline__ int place_of(u64 key) { return (int)~(unsigned)key; }

// what a CTA shows the others of its cluster
struct Board {
    float m, s, w;
    int n;                    // keys in `best`
    u64 best[MAX_TOP];        // descending
};

struct Shared {
    uint4 ring[RING];
    unsigned long long full[8], empty[8];
    Board board;
    u64 notes[NOTES];
    u64 groups[GROUPS];
    u64 bound;
    int n_notes, lost;        // lost: a note did not fit
    float red[3][THREADS / 32];
};

__device__ int g_error = 0;
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, int code) { return sm100::mbar_wait_bounded(bar, parity, &g_error, code); }

// the threads that look at logits meet; whether any of them has `mine`
__device__ __forceinline__ bool meet(bool mine) {
    int any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((int)mine) : "memory");
    return any != 0;
}
static_assert(THREADS == 256, "the barrier's number of threads");

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int remote_i32(const int* local, unsigned rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(ib_cluster_address(local, rank)));
    return v;
}
__device__ __forceinline__ u64 remote_u64(const u64* local, unsigned rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(ib_cluster_address(local, rank)));
    return v;
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// S and W from reference m to reference to >= m (S = W = 0 where m is minus infinity)
__device__ __forceinline__ void move_reference(float m, float to, float& s, float& w) {
    if (m == to || m == -INFINITY) return;
    const float g = (m - to) * LOG2E, c = sm100::ex2(g);
    w = c > 0.0f ? c * fmaf(s, g, w) : 0.0f;
    s *= c;
}

// two neighbouring numbers at once
__device__ __forceinline__ u64 pair(float a, float b) {
    u64 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void apart(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// the logits e, the largest of which is `top`, to a thread's m, S and W
template <int EACH>
__device__ __forceinline__ void add_block(const float* e, float top, float& m, float& s, float& w) {
    if (top > m) {
        move_reference(m, top, s, w);
        m = top;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    const u64 less = pair(-ref, -ref), factor = pair(LOG2E, LOG2E);
    u64 s2 = 0, w2 = 0;
#pragma unroll
    for (int i = 0; i < EACH; i += 2) {
        float a, b;
        apart(mul2(add2(pair(e[i], e[i + 1]), less), factor), a, b);       // (log2(e) z; the difference is taken first: large logits lose nothing)
        a = fmaxf(a, LOWEST);
        b = fmaxf(b, LOWEST);
        const u64 p = pair(sm100::ex2(a), sm100::ex2(b));
        s2 = add2(s2, p);
        w2 = fma2(p, pair(a, b), w2);
    }
    float a, b;
    apart(s2, a, b);
    s += a + b;
    apart(w2, a, b);
    w += a + b;
}

// The k best of the first n notes to best[0 .. min(k, n)) in descending order, by counting the keys ahead of each (keys differ:
// they hold their places), four threads a key where there are few.  The threads that look at logits call it between two meetings.
__device__ __noinline__ void rank_notes(const u64* notes, int n, int k, u64* best) {
    const int log = n <= THREADS / 4 ? 2 : 0, share = 1 << log, part = threadIdx.x & (share - 1);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += THREADS >> log) {
        const int i = i0 + (threadIdx.x >> log);
        const u64 mine = i < n ? notes[i] : ~0ull;
        int ahead = 0;
#pragma unroll 4
        for (int j = part; j < n; j += share) ahead += notes[j] > mine;
        if (share == 4) {
            ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
            ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
        }
        if (i < n && part == 0 && ahead < k) best[ahead] = mine;
    }
}

struct Args {
    const void* logits;
    const int* tokens;
    float* log_probs;
    float* entropy;
    int* top_ids;
    float* top_log_probs;
    long ld;
    int rows, vocab, given, top;
};

template <typename T> struct Wide;      // logits of a vector, vectors of a thread's share of a chunk
template <> struct Wide<float> {
    static constexpr int N = 4, VECTORS = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <> struct Wide<__nv_bfloat16> {
    static constexpr int N = 8, VECTORS = 2;
    static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
        const unsigned r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r[i] << 16);
            x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS + 32, 3) log_probs_kernel(const Args A, int cluster) {
    constexpr int N = Wide<T>::N, VECTORS = Wide<T>::VECTORS, EACH = N * VECTORS;      // logits that a thread takes at once
    constexpr int CHUNK = THREADS * VECTORS, STAGES = RING / CHUNK;
    static_assert(STAGES <= 8, "");
    extern __shared__ __align__(128) unsigned char raw[];
    Shared& sh = *reinterpret_cast<Shared*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / cluster;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const T* x = static_cast<const T*>(A.logits) + (long)row * A.ld;
    // this CTA's stretch of the row: vectors v_lo .. v_hi, counted from the 16-byte boundary at or before the row's start
    const int skew = (int)(((unsigned long long)x / sizeof(T)) % N);
    const int vectors = (A.vocab + skew + N - 1) / N;
    const int v_lo = (int)((long)vectors * rank / cluster), v_hi = (int)((long)vectors * (rank + 1) / cluster);
    // the whole ones among them; at the row's ends a vector may hold what is not the row's
    const int w_lo = v_lo == 0 && skew ? 1 : v_lo, w_hi = min(v_hi, (A.vocab + skew) / N);
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            sm100::mbar_init(sm100::smem_u32(&sh.full[s]), 1);
            sm100::mbar_init(sm100::smem_u32(&sh.empty[s]), THREADS / 32);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.n_notes = sh.lost = 0;
    }
    __syncthreads();

    float m = -INFINITY, s = 0.0f, w = 0.0f;
    u64 bound = 0;                    // keys below it are not noted
    float least = -INFINITY;          // its value
    const int rounds = (v_hi - v_lo + CHUNK - 1) / CHUNK;
    int round = 0, next_look = 2;
    bool ok = true;
    auto note = [&](u64 key) {
        const int at = atomicAdd(&sh.n_notes, 1);
        if (at < NOTES) sh.notes[at] = key;
        else sh.lost = 1;
    };
    // the k best of what is noted take its place and give the next bound (the threads have met)
    auto prune = [&]() {
        const int n = min(sh.n_notes, NOTES);
        rank_notes(sh.notes, n, A.top, sh.board.best);
        meet(false);
        const int left = min(n, A.top);
        if (tid < left) sh.notes[tid] = sh.board.best[tid];
        if (tid == 0) sh.n_notes = left;
        if (left == A.top) {
            bound = max(bound, sh.board.best[A.top - 1]);
            least = value_of(bound);
        }
        meet(false);
    };
    // the given tokens' logits, on their way meanwhile
    float given = -INFINITY;
    if (rank == 0 && tid < A.given) {
        const int t = A.tokens[(long)row * A.given + tid];
        if (t >= 0 && t < A.vocab) given = fmaxf(ib_to_float(x[t]), -INFINITY);
    }
    if (warp == THREADS / 32) {       // the logits come as bulk copies: three CTAs of an SM have up to 192 KB on their way
        if (lane == 0) {
            for (int v0 = v_lo; v0 < v_hi && ok; v0 += CHUNK, ++round) {
                const int stage = round % STAGES;
                if (round >= STAGES) ok = mbar_wait(sm100::smem_u32(&sh.empty[stage]), (round / STAGES - 1) & 1, 1);
                if (!ok) break;
                const int from = max(v0, w_lo), to = min(v0 + CHUNK, w_hi);
                const unsigned bytes = to > from ? (unsigned)(to - from) * 16u : 0u, full = sm100::smem_u32(&sh.full[stage]);
                sm100::mbar_expect_tx(full, bytes);
                if (bytes)
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(sm100::smem_u32(&sh.ring[stage * CHUNK + from - v0])), "l"(x + ((long)from * N - skew)), "r"(bytes), "r"(full) : "memory");
            }
        }
        __syncwarp();
    } else
    for (int v0 = v_lo; v0 < v_hi; v0 += CHUNK, ++round) {
        const int stage = round % STAGES;
        if (ok && !mbar_wait(sm100::smem_u32(&sh.full[stage]), (round / STAGES) & 1, 2)) ok = false;
        float e[EACH];
        // (a thread's vectors are neighbours; in an order of its own, so that eight threads' meet all banks)
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) Wide<T>::unpack(sh.ring[stage * CHUNK + tid * VECTORS + ((i + lane / (8 / VECTORS)) & (VECTORS - 1))], e + i * N);
        if (v0 < w_lo || v0 + CHUNK > w_hi) {      // at a row's ends some vectors are not whole
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                const int v = v0 + tid * VECTORS + ((i + lane / (8 / VECTORS)) & (VECTORS - 1));
                if (v >= w_lo && v < w_hi) continue;
#pragma unroll
                for (int c = 0; c < N; ++c) {
                    const int at = v * N - skew + c;
                    e[i * N + c] = v < v_hi && at >= 0 && at < A.vocab ? ib_to_float(x[at]) : NAN;
                }
            }
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(&sh.empty[stage]));
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i) top = fmaxf(top, e[i]);
        add_block<EACH>(e, top, m, s, w);
        if constexpr (TOP) {
            auto key = [&]() -> u64 {      // (a logit of minus infinity is one, no number is none)
                bool any = top > -INFINITY;
                if (!any) {
#pragma unroll
                    for (int i = 0; i < EACH; ++i) any |= e[i] == e[i];
                }
                return any ? key_of(top, v0 + tid * VECTORS) : 0;
            };
            if (round == 0) {      // the first bound
                u64 best = key();
#pragma unroll
                for (int o = 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
                if ((tid & 3) == 0) sh.groups[tid >> 2] = best;
                meet(false);
                const int group = tid >> 2;
                const u64 mine = sh.groups[group];
                int ahead = 0;
#pragma unroll 8
                for (int j = tid & 3; j < GROUPS; j += 4) ahead += sh.groups[j] > mine || (sh.groups[j] == mine && j < group);
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
                if ((tid & 3) == 0 && ahead == A.top - 1) sh.bound = mine;       // (0 where fewer groups hold a number)
                meet(false);
                bound = sh.bound;
                if (bound) least = value_of(bound);
            }
            if (top >= least) {
                const u64 mine = key();
                if (mine >= bound && mine) note(mine);
            }
            if (round == next_look) {      // (not when few logits are to come: the last look is near)
                if (3 * round < rounds) {
                    meet(false);
                    prune();
                }
                next_look = 2 * round + 1;
            }
        }
    }
    __syncthreads();
    if (TOP && tid < THREADS) {
        auto logit = [&](int v, int c) {       // logit c of the block that starts with vector v
            const int at = v * N - skew + c;
            return v + c / N < v_hi && at >= 0 && at < A.vocab ? ib_to_float(x[at]) : NAN;
        };
        if (sh.lost) {
            // More notes than there is room for (logits that ascend do that): from the best bound so far on, the blocks again, with a look whenever
            // the room could run out.  Nothing is lost then.
            meet(false);
            prune();
            if (tid == 0) sh.n_notes = 0;
            meet(false);
            for (int v0 = v_lo; v0 < v_hi; v0 += CHUNK) {
                const int v = v0 + tid * VECTORS;
                float top = -INFINITY;
                bool any = false;
                for (int c = 0; c < EACH; ++c) {
                    const float z = logit(v, c);
                    top = fmaxf(top, z);
                    any |= z == z;
                }
                if (any && key_of(top, v) >= bound) note(key_of(top, v));
                meet(false);
                const bool look = sh.n_notes > NOTES - THREADS;
                meet(false);
                if (look) prune();
            }
            meet(false);
        }
        // the k best blocks' logits: those that reach the k-th block's largest one
        prune();
        const int blocks = sh.n_notes;
        if (blocks < A.top) least = -INFINITY;
        meet(false);
        if (tid == 0) sh.n_notes = 0;
        meet(false);
        for (int i = tid; i < blocks * EACH; i += THREADS) {
            const int v = place_of(sh.board.best[i / EACH]), c = i % EACH;
            const float z = logit(v, c);
            if (z >= least) note(key_of(z, v * N - skew + c));      // (at most 512: there is room)
        }
        meet(false);
        rank_notes(sh.notes, sh.n_notes, A.top, sh.groups);
        meet(false);
        if (tid < A.top) sh.board.best[tid] = sh.groups[tid];
        if (tid == 0) sh.n_notes = min(sh.n_notes, A.top);
    }

    // the CTA's m, S and W
    float top = ib_warp_max(m);
    move_reference(m, top, s, w);
    s = ib_warp_sum(s);
    w = ib_warp_sum(w);
    if (lane == 0 && warp < THREADS / 32) { sh.red[0][warp] = top; sh.red[1][warp] = ok ? s : NAN; sh.red[2][warp] = w; }
    __syncthreads();
    if (warp == 0) {
        const int n = THREADS / 32;
        float m1 = lane < n ? sh.red[0][lane] : -INFINITY, s1 = lane < n ? sh.red[1][lane] : 0.0f, w1 = lane < n ? sh.red[2][lane] : 0.0f;
        const float all = ib_warp_max(m1);
        move_reference(m1, all, s1, w1);
        s1 = ib_warp_sum(s1);
        w1 = ib_warp_sum(w1);
        if (lane == 0) {
            sh.board.m = all; sh.board.s = s1; sh.board.w = w1;
            sh.board.n = TOP ? sh.n_notes : 0;
        }
    }
    if (cluster > 1) ib_cluster_sync(); else __syncthreads();
    if (rank == 0) {
        // lane c looks at the c-th CTA's sums; all warps add them in the same order
        float mc = -INFINITY, total = 0.0f, weighed = 0.0f;
        int have = 0;
        if (lane < cluster) {
            mc = ib_cluster_f32(&sh.board.m, lane);
            total = ib_cluster_f32(&sh.board.s, lane);
            weighed = ib_cluster_f32(&sh.board.w, lane);
            have = remote_i32(&sh.board.n, lane);
        }
        const float all = ib_warp_max(mc);
        move_reference(mc, all, total, weighed);
#pragma unroll
        for (int o = IB_MAX_CLUSTER / 2; o > 0; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            weighed += __shfl_xor_sync(0xffffffffu, weighed, o);
            have += __shfl_xor_sync(0xffffffffu, have, o);
        }
        total = __shfl_sync(0xffffffffu, total, 0);
        weighed = __shfl_sync(0xffffffffu, weighed, 0);
        have = __shfl_sync(0xffffffffu, have, 0);
        const bool none = !(fabsf(all) < INFINITY);
        const float log_total = none ? NAN : logf(total);
        if (tid == 0 && A.entropy) A.entropy[row] = log_total - LN2 * (weighed / total);
        for (int i = tid; i < A.given; i += THREADS + 32) {
            float v = given;
            if (i != tid) {
                const int t = A.tokens[(long)row * A.given + i];
                v = t >= 0 && t < A.vocab ? fmaxf(ib_to_float(x[t]), -INFINITY) : -INFINITY;
            }
            A.log_probs[(long)row * A.given + i] = (v - all) - log_total;
        }
        if constexpr (TOP) {
            if (cluster > 1) {      // the best of the CTAs' best
                const int all_keys = cluster * A.top, of = tid / A.top, i = tid - of * A.top;
                u64 mine = 0;
                const int theirs = tid < all_keys ? remote_i32(&sh.board.n, of) : 0;
                if (i < theirs) mine = remote_u64(&sh.board.best[i], of);
                if (tid < all_keys) sh.notes[tid] = mine;
                __syncthreads();
                if (mine) {
                    int ahead = 0;
#pragma unroll 8
                    for (int j = 0; j < all_keys; ++j) ahead += sh.notes[j] > mine;
                    if (ahead < A.top) {
                        A.top_ids[(long)row * A.top + ahead] = place_of(mine);
                        A.top_log_probs[(long)row * A.top + ahead] = (value_of(mine) - all) - log_total;
                    }
                }
                for (int i = have + tid; i < A.top; i += THREADS + 32) {
                    A.top_ids[(long)row * A.top + i] = -1;
                    A.top_log_probs[(long)row * A.top + i] = -INFINITY;
                }
            } else {
                for (int i = tid; i < A.top; i += THREADS + 32) {
                    const bool some = i < sh.board.n;
                    A.top_ids[(long)row * A.top + i] = some ? place_of(sh.board.best[i]) : -1;
                    A.top_log_probs[(long)row * A.top + i] = some ? (value_of(sh.board.best[i]) - all) - log_total : -INFINITY;
                }
            }
        }
    }
    if (cluster > 1) ib_cluster_sync();        // nobody leaves while rank 0 reads
}

// The same with a warp a row, for many rows of few logits: a lane takes every 32nd block of 16, all of whose keys stay in its registers.  The likeliest
// tokens come one by one: the block with the best key is looked at by 16 lanes, and its next logit's key takes that one's place.
constexpr int LANE_BLOCKS = 16, SHORT = LANE_BLOCKS * 512;      // a lane's blocks at most; logits of a row, counted from the 16-byte boundary

__device__ __forceinline__ u64 warp_best(u64 key) {
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
    return (u64)high << 32 | __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32) == high ? (unsigned)key : 0u);
}

template <typename T, bool TOP, int BLOCKS>
__global__ void __launch_bounds__(128) short_rows_kernel(const Args A) {
    constexpr int N = Wide<T>::N, VECTORS = Wide<T>::VECTORS, EACH = N * VECTORS;
    static_assert(EACH == 16, "");
    const int lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= A.rows) return;
    const T* x = static_cast<const T*>(A.logits) + row * A.ld;
    const int skew = (int)(((unsigned long long)x / sizeof(T)) % N), end = A.vocab + skew;      // places are counted from the boundary
    const T* from = x - skew;
    float m = -INFINITY, s = 0.0f, w = 0.0f;
    u64 keys[BLOCKS];
    uint4 next[VECTORS];
    auto fetch = [&](int place) {
        if (place >= skew && place + EACH <= end)
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) next[i] = *reinterpret_cast<const uint4*>(from + place + i * N);
    };
    fetch(lane * EACH);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        keys[b] = 0;
        if (b * 32 * EACH >= end) continue;
        const int place = (b * 32 + lane) * EACH;
        float e[EACH];
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) Wide<T>::unpack(next[i], e + i * N);
        if (place < skew || place + EACH > end) {
#pragma unroll
            for (int c = 0; c < EACH; ++c) e[c] = place + c >= skew && place + c < end ? ib_to_float(from[place + c]) : NAN;
        }
        fetch(place + 32 * EACH);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i) top = fmaxf(top, e[i]);
        bool any = top > -INFINITY;        // (a logit of minus infinity is one, no number is none)
        if (TOP && !any) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) any |= e[i] == e[i];
        }
        add_block<EACH>(e, top, m, s, w);
        if (TOP && any) keys[b] = key_of(top, place);
    }
    const float all = ib_warp_max(m);
    move_reference(m, all, s, w);
    s = ib_warp_sum(s);
    w = ib_warp_sum(w);
    const bool none = !(fabsf(all) < INFINITY);
    const float log_total = none ? NAN : logf(s);
    if (lane == 0 && A.entropy) A.entropy[row] = log_total - LN2 * (w / s);
    for (int i = lane; i < A.given; i += 32) {
        const int t = A.tokens[row * A.given + i];
        const float v = t >= 0 && t < A.vocab ? fmaxf(ib_to_float(x[t]), -INFINITY) : -INFINITY;
        A.log_probs[row * A.given + i] = (v - all) - log_total;
    }
    if constexpr (TOP) {
        u64 mine = 0;                      // the lane-th likeliest
#pragma unroll 1
        for (int i = 0; i < A.top; ++i) {
            u64 best = 0;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) best = max(best, keys[b]);
            best = warp_best(best);
            if (best == 0) break;
            // a block's key is that of a logit that comes next, or, before the first one was taken, no less than its largest logit's
            const int block = place_of(best) / EACH, place = block * EACH + (lane & (EACH - 1));
            u64 key = 0;
            if (place >= skew && place < end) {
                const float z = ib_to_float(from[place]);
                key = z == z ? key_of(z, place) : 0;
            }
            if (key > best) key = 0;
            const u64 first = warp_best(key), second = warp_best(key == first ? 0 : key);
            if (lane == i) mine = first;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
                if (b * 32 + lane == block) keys[b] = second;
        }
        if (lane < A.top) {
            A.top_ids[row * A.top + lane] = mine ? place_of(mine) - skew : -1;
            A.top_log_probs[row * A.top + lane] = mine ? (value_of(mine) - all) - log_total : -INFINITY;
        }
    }
}

template <typename T, bool TOP>
static int launch(const Args& a, bool short_rows, cudaStream_t stream) {
    if (short_rows) {
        const unsigned grid = (unsigned)((a.rows + 3L) / 4);
        if (a.vocab + 7 <= SHORT / 2) short_rows_kernel<T, TOP, LANE_BLOCKS / 2><<<grid, 128, 0, stream>>>(a);
        else short_rows_kernel<T, TOP, LANE_BLOCKS><<<grid, 128, 0, stream>>>(a);
        return ib_launch_status();
    }
    static IbDeviceSet done;
    if (const int code = ib_allow_dynamic_smem(done, log_probs_kernel<T, TOP>, sizeof(Shared))) return code;
    // As many CTAs for a row as the machine has room for (three on each of 148 SMs, clusters that run at once), each with at least a chunk's logits.
    // (1, 2, 4, 8 CTAs a row, the five most likely tokens: 128 rows of 151,936 logits 30, 22.5, 29, 36 us; one row 28, 18.8, 13.4, 10.1; one of 16,384
    // 8.0, 7.8, 7.2, 7.4; one of 4,000 6.2, 7.1, 7.2, 7.2.  50 rows, whose clusters of eight take two turns, 21.1, of four 15.7.)
    static IbClusters clusters;
    int cluster = 1;
    while (cluster < IB_MAX_CLUSTER && (long)a.rows * cluster * 2 <= 444 && a.vocab >= 4096L * cluster * 2) cluster *= 2;
    while (cluster > 1 && ib_clusters_at_once(clusters, log_probs_kernel<T, TOP>, cluster, THREADS + 32, sizeof(Shared)) < a.rows) cluster /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.gridDim = dim3((unsigned)(a.rows * cluster));
    cfg.blockDim = dim3(THREADS + 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, log_probs_kernel<T, TOP>, a, cluster);
    return ib_launch_status();
}

}  // namespace lp

struct IbTokenLogProbs {
    const void* logits;
    const int* tokens;
    float *log_probs, *entropy;
    int* top_ids;
    float* top_log_probs;
    cudaStream_t stream;
    long f32, ld, rows, vocab, given, top;
};

IB_EXPORT int ib_token_log_probs(const void* call) {
    using namespace lp;
    const IbTokenLogProbs c = *static_cast<const IbTokenLogProbs*>(call);
    if (c.rows < 0 || c.vocab <= 0 || c.given < 0 || c.top < 0) return IB_ERR_ARGUMENT;
    if (c.top > MAX_TOP || c.vocab > 0x40000000L || c.rows > 0x7fffffffL / IB_MAX_CLUSTER || c.given > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    if (c.rows == 0) return IB_OK;
    const Args a{c.logits, c.tokens, c.log_probs, c.entropy, c.top_ids, c.top_log_probs, c.ld, (int)c.rows, (int)c.vocab, (int)c.given, (int)c.top};
    // A warp for a row of few logits where there are more rows than the SMs hold CTAs, or few logits and few tokens wanted of them.  (A CTA and a
    // warp a row: 4,096 rows of 1,000 with the five likeliest 60.6 and 10.1 us, of 8,000 73 and 39; 500 rows of 8,000 13.8 and 10.9, with 32
    // 18.2 and 18.9; 300 rows of 1,000 8.2 and 4.7, of 8,000 9.0 and 10.9, of 1,000 with 32 9.3 and 10.9.)
    const bool short_rows = c.vocab + 7 <= SHORT && (c.rows > 444 || (c.vocab <= 2048 && c.top <= 8));
    if (c.f32) return c.top ? launch<float, true>(a, short_rows, c.stream) : launch<float, false>(a, short_rows, c.stream);
    return c.top ? launch<__nv_bfloat16, true>(a, short_rows, c.stream) : launch<__nv_bfloat16, false>(a, short_rows, c.stream);
}

IB_EXPORT int ib_log_probs_error(int reset) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, lp::g_error, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(lp::g_error, &zero, sizeof(int));
    }
    return v;
}
IB_EXPORT int ib_log_probs_error_async(int* out, cudaStream_t stream) {
    return (int)cudaMemcpyFromSymbolAsync(out, lp::g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}
