// Log probabilities of given tokens, the distribution's entropy and its most likely tokens, for every row of logits.
//
// With m the row's largest logit, z = x - m, S = sum e^z and W = sum e^z z:
//   log p(t) = z_t - log S        entropy = -sum p log p = log S - W / S
// S and W are sums of numbers of one sign and lose nothing to cancellation.  Every thread keeps m, S and W of what it has seen
// in 32 bits; when its m grows by g, S becomes S e^-g and W becomes (W - S g) e^-g.  A logit that is no number counts as minus
// infinity, as it does for the sampler; a row whose largest logit is infinite has no distribution, and NaN as its numbers.
//
// The logits are read once.  The k most likely tokens come out of the same pass: a key is the logit's bits made ascending, the
// place's complement below them (of equal logits the lower place is ahead).  A bound that at least k keys of the row reach is
// kept; what passes it is noted in shared memory, and now and then the k best of the noted ones give a higher bound.  The first
// bound is the k-th largest of 64 groups' largest keys; expected are k to 2 k notes from the first 8,192 logits and k more
// for every doubling behind them.
#include "common.cuh"

namespace lp {

constexpr int THREADS = 512;
constexpr int MAX_TOP = 32;
constexpr int NOTES = 1024;          // room for noted keys
constexpr int GROUPS = 64;           // groups of 8 threads whose largest keys give the first bound
constexpr int MAX_CLUSTER = 8;
constexpr float LOWEST = -200.0f;    // e^-200 is 0 in 32 bits, and 0 times it is 0

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
    Board board;
    u64 notes[NOTES];
    u64 groups[GROUPS];
    u64 bound;
    int n_notes;
    float red[3][THREADS / 32];
};

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned remote(const void* local, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ float remote_f32(const float* local, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int remote_i32(const int* local, unsigned rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 remote_u64(const u64* local, unsigned rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(local, rank)) : "memory");
    return v;
}

// S and W from reference m to reference to >= m (S = W = 0 where m is minus infinity)
__device__ __forceinline__ void move_reference(float m, float to, float& s, float& w) {
    if (m == to || m == -INFINITY) return;
    const float g = m - to;
    const float c = __expf(g);
    w = c > 0.0f ? c * fmaf(s, g, w) : 0.0f;
    s *= c;
}

// The k best of the first n notes to best[0 .. min(k, n)) in descending order, by counting the keys ahead of each (keys differ:
// they hold their places).  The whole CTA calls it between two barriers.
__device__ __forceinline__ void rank_notes(const u64* notes, int n, int k, u64* best) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const u64 mine = notes[i];
        int ahead = 0;
        for (int j = 0; j < n; ++j) ahead += notes[j] > mine;
        if (ahead < k) best[ahead] = mine;
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

template <typename T> struct Wide;
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
__global__ void __launch_bounds__(THREADS, 2) log_probs_kernel(const Args A, int cluster) {
    constexpr int N = Wide<T>::N, VECTORS = Wide<T>::VECTORS, EACH = N * VECTORS;      // logits that a thread takes at once
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / cluster;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const T* x = static_cast<const T*>(A.logits) + (long)row * A.ld;
    // this CTA's stretch [lo, hi), cut on whole vectors counted from the 16-byte boundary at or before the row's start
    const int skew = (int)(((unsigned long long)x / sizeof(T)) % N);
    const int vectors = (A.vocab + skew + N - 1) / N;
    const int v_lo = (int)((long)vectors * rank / cluster), v_hi = (int)((long)vectors * (rank + 1) / cluster);
    const int hi = min(A.vocab, v_hi * N - skew), lo = max(0, v_lo * N - skew);

    float m = -INFINITY, s = 0.0f, w = 0.0f;
    u64 bound = 0;                    // keys below it are not noted
    float bound_v = -INFINITY;
    if (TOP && tid == 0) sh.n_notes = 0;
    int round = 0, next_look = 2;
    for (int v0 = v_lo; v0 < v_hi; v0 += THREADS * VECTORS, ++round) {
        float e[EACH];
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) {
            const int at = (v0 + i * THREADS + tid) * N - skew;
            if (at >= lo && at + N <= hi) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(x + at));
                Wide<T>::unpack(v, e + i * N);
            } else {
#pragma unroll
                for (int c = 0; c < N; ++c) e[i * N + c] = at + c >= lo && at + c < hi ? ib_to_float(x[at + c]) : NAN;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i) top = fmaxf(top, e[i]);
        if (top > m) {
            move_reference(m, top, s, w);
            m = top;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const float z = fmaxf(e[i] - ref, LOWEST);
            const float p = __expf(z);
            s += p;
            w = fmaf(p, z, w);
        }
        if constexpr (TOP) {
            auto place = [&](int i) { return (v0 + (i / N) * THREADS + tid) * N - skew + i % N; };
            if (round == 0) {      // the first bound
                u64 best = 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                    if (e[i] == e[i]) best = max(best, key_of(e[i], place(i)));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
                if ((tid & 7) == 0) sh.groups[tid >> 3] = best;
                __syncthreads();
                if (tid < GROUPS) {
                    const u64 mine = sh.groups[tid];
                    int ahead = 0;
                    for (int j = 0; j < GROUPS; ++j) ahead += sh.groups[j] > mine || (sh.groups[j] == mine && j < tid);
                    if (ahead == A.top - 1) sh.bound = mine;       // (0 where fewer groups hold a number)
                }
                __syncthreads();
                bound = sh.bound;
                bound_v = bound ? value_of(bound) : -INFINITY;
            }
            unsigned todo = 0;
            if (top >= bound_v) {
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                    if (e[i] >= bound_v && key_of(e[i], place(i)) >= bound) todo |= 1u << i;
            }
            for (;;) {
                bool full = false;
                if (todo) {
#pragma unroll
                    for (int i = 0; i < EACH; ++i) {
                        if (!(todo >> i & 1) || full) continue;
                        const u64 key = key_of(e[i], place(i));
                        if (key >= bound) {
                            const int at = atomicAdd(&sh.n_notes, 1);
                            if (at < NOTES) sh.notes[at] = key; else full = true;
                        }
                        if (!full) todo &= ~(1u << i);
                    }
                }
                const bool again = __syncthreads_or(full);
                if (!again && round < next_look) break;
                // the k best of what is noted take its place and give the next bound
                const int n = min(sh.n_notes, NOTES);
                rank_notes(sh.notes, n, A.top, sh.board.best);
                __syncthreads();
                const int left = min(n, A.top);
                if (tid < left) sh.notes[tid] = sh.board.best[tid];
                if (tid == 0) sh.n_notes = left;
                if (left == A.top) {
                    bound = max(bound, sh.board.best[A.top - 1]);
                    bound_v = bound ? value_of(bound) : -INFINITY;
                }
                __syncthreads();
                if (!again) { next_look = 2 * round + 1; break; }
            }
        }
    }

    // the CTA's m, S and W
    float top = ib_warp_max(m);
    move_reference(m, top, s, w);
    s = ib_warp_sum(s);
    w = ib_warp_sum(w);
    if (lane == 0) { sh.red[0][warp] = top; sh.red[1][warp] = s; sh.red[2][warp] = w; }
    __syncthreads();
    if (TOP) rank_notes(sh.notes, min(sh.n_notes, NOTES), A.top, sh.board.best);
    if (warp == 0) {
        const int n = THREADS / 32;
        float m1 = lane < n ? sh.red[0][lane] : -INFINITY, s1 = lane < n ? sh.red[1][lane] : 0.0f, w1 = lane < n ? sh.red[2][lane] : 0.0f;
        const float all = ib_warp_max(m1);
        move_reference(m1, all, s1, w1);
        s1 = ib_warp_sum(s1);
        w1 = ib_warp_sum(w1);
        if (lane == 0) {
            sh.board.m = all; sh.board.s = s1; sh.board.w = w1;
            sh.board.n = TOP ? min(min(sh.n_notes, NOTES), A.top) : 0;
        }
    }
    if (cluster > 1) cluster_sync(); else __syncthreads();
    if (rank == 0) {
        // every thread adds the CTAs' sums in the same order
        float all = -INFINITY, total = 0.0f, weighed = 0.0f;
        for (int c = 0; c < cluster; ++c) all = fmaxf(all, cluster > 1 ? remote_f32(&sh.board.m, c) : sh.board.m);
        for (int c = 0; c < cluster; ++c) {
            float sc = cluster > 1 ? remote_f32(&sh.board.s, c) : sh.board.s, wc = cluster > 1 ? remote_f32(&sh.board.w, c) : sh.board.w;
            move_reference(cluster > 1 ? remote_f32(&sh.board.m, c) : sh.board.m, all, sc, wc);
            total += sc;
            weighed += wc;
        }
        const bool none = !(fabsf(all) < INFINITY);
        const float log_total = none ? NAN : logf(total);
        if (tid == 0 && A.entropy) A.entropy[row] = log_total - weighed / total;
        for (int i = tid; i < A.given; i += THREADS) {
            const int t = A.tokens[(long)row * A.given + i];
            float v = -INFINITY;
            if (t >= 0 && t < A.vocab) v = fmaxf(ib_to_float(x[t]), -INFINITY);
            A.log_probs[(long)row * A.given + i] = (v - all) - log_total;
        }
        if constexpr (TOP) {
            if (cluster > 1) {      // the best of the CTAs' best
                u64 mine = 0;
                int of = 0;
                if (tid < cluster * MAX_TOP) {
                    of = tid / MAX_TOP;
                    const int i = tid % MAX_TOP;
                    if (i < remote_i32(&sh.board.n, of)) mine = remote_u64(&sh.board.best[i], of);
                    sh.notes[tid] = mine;
                }
                __syncthreads();
                if (tid < cluster * MAX_TOP && mine) {
                    int ahead = 0;
                    for (int j = 0; j < cluster * MAX_TOP; ++j) ahead += sh.notes[j] > mine;
                    if (ahead < A.top) {
                        A.top_ids[(long)row * A.top + ahead] = place_of(mine);
                        A.top_log_probs[(long)row * A.top + ahead] = (value_of(mine) - all) - log_total;
                    }
                }
                int have = 0;
                for (int c = 0; c < cluster; ++c) have += remote_i32(&sh.board.n, c);
                for (int i = have + tid; i < A.top; i += THREADS) {
                    A.top_ids[(long)row * A.top + i] = -1;
                    A.top_log_probs[(long)row * A.top + i] = -INFINITY;
                }
            } else {
                for (int i = tid; i < A.top; i += THREADS) {
                    const bool some = i < sh.board.n;
                    A.top_ids[(long)row * A.top + i] = some ? place_of(sh.board.best[i]) : -1;
                    A.top_log_probs[(long)row * A.top + i] = some ? (value_of(sh.board.best[i]) - all) - log_total : -INFINITY;
                }
            }
        }
    }
    if (cluster > 1) cluster_sync();        // nobody leaves while rank 0 reads
}

template <typename T, bool TOP>
static int launch(const Args& a, int cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * cluster));
    cfg.blockDim = dim3(THREADS);
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
    if (c.top > MAX_TOP || c.vocab > 0x40000000L || c.rows > 0x7fffffffL / MAX_CLUSTER || c.given > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    if (c.rows == 0) return IB_OK;
    const Args a{c.logits, c.tokens, c.log_probs, c.entropy, c.top_ids, c.top_log_probs, c.ld, (int)c.rows, (int)c.vocab, (int)c.given, (int)c.top};
    // as many CTAs for a row as the machine has room for (two on each of 148 SMs), each with at least 4,096 logits
    int cluster = 1;
    while (cluster < MAX_CLUSTER && c.rows * cluster * 2 <= 296 && c.vocab >= 4096L * cluster * 2) cluster *= 2;
    if (c.f32) return c.top ? launch<float, true>(a, cluster, c.stream) : launch<float, false>(a, cluster, c.stream);
    return c.top ? launch<__nv_bfloat16, true>(a, cluster, c.stream) : launch<__nv_bfloat16, false>(a, cluster, c.stream);
}
