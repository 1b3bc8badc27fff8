// Log-probabilities of given items under the softmax over a whole catalog, with the entropy and the K best items, and
// their gradient.  For a row x of V logits (M = max x, Z = sum exp(x - M)):
//   logp_t = (x_t - M) - log Z       H = log Z - (sum exp(x - M) (x - M)) / Z
//   dx_v = sum_t g_t [v = t] - p_v (sum_t g_t + gH (log p_v + H)),   p_v = exp(x_v - M) / Z
// HBM-bound: the forward reads the logits once (running maximum and sums per lane, rescaled when the maximum moves), the
// gradient reads them once and writes once.  M and log Z are kept apart: with logits of 10^4, M + log Z has lost the
// digits that p needs.
//
// A wavefront works alone: its lanes' 16-byte pieces, its statistics and its list of candidates for the K best, so the
// loop has no workgroup barrier.  Candidates cost nothing on the way: a group of pieces is looked at only if its maximum
// (needed anyway) reaches the wavefront's threshold, which starts at the K-th best of the lanes' first maxima -- a
// lower bound of the K-th best -- and rises whenever the list of 256 is cut back to K.
//   V <= 2048, or at least 2048 rows of up to 16384   one wavefront per row: nothing to join.  Forward of 4096 x 3707 fp16:
//                            11.7 us, 18.2 us with a workgroup per row; of 4096 x 1000 with K = 10: 10 and 28 us; but of
//                            1024 x 8000 fp32 with K = 10: 22.0 us, 17.3 us with a workgroup per row
//   many longer rows         one workgroup of 4 wavefronts per row
//   few rows                 the row is split over workgroups; logp_join_kernel adds up their parts
// Forward of 4096 x 100000 fp32 with K = 10: 318 us a call, back to back, = 5.2 TB/s (333 - 338 us under the profiler); gradient
// of 4096 x 30000 bf16: 105 us = 4.7 TB/s.
#include "dr_types.h"

namespace dr {

constexpr int LP_MAX_K = 64, LP_MAX_T = 64;
constexpr int LP_CAP = 256;        // candidates of a wavefront
constexpr int LP_MAX_SPLITS = 256;
constexpr int64_t LP_MAX_GRID = 1 << 24;   // workgroups of 256: a launch counts its threads in 32 bits
constexpr float LP_LOG2E = 1.44269504088896340736f;
constexpr float LP_LOWEST = -3.402823466e38f;
constexpr float LP_FLOOR = -200.0f;   // exp(-200) is 0 in fp32: keeps 0 * -inf out of the entropy sum

struct LogpArgs {
    const void* x;
    int64_t ld, N;
    int V;
    const void* tgt;
    int id64, T, K;
    int splits, seg;          // workgroups per row, elements each
    float *logp, *ent, *lse;  // lse [N, 2]: M, log Z
    int32_t* top_idx;
    float* top_logp;
    float* pst;               // [N, splits, 4] M, Z, sum
    uint64_t* pkey;           // [N, splits, 4, K]
};

// ---- (M, Z, S = sum exp(x - M) (x - M)) ----------------------------------------------------------------------------
struct Stat {
    float m, z, s;
};
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }
__device__ __forceinline__ Stat stat_join(const Stat& a, const Stat& b) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m, ea = lp_exp(da), eb = lp_exp(db);
    r.z = a.z * ea + b.z * eb;
    r.s = ea * (a.s + a.z * fmaxf(da, LP_FLOOR)) + eb * (b.s + b.z * fmaxf(db, LP_FLOOR));
    return r;
}
__device__ __forceinline__ Stat stat_wave(Stat a) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        Stat b;
        b.m = __shfl_xor(a.m, off, 64);
        b.z = __shfl_xor(a.z, off, 64);
        b.s = __shfl_xor(a.s, off, 64);
        a = stat_join(a, b);
    }
    return a;
}

// ---- candidates for the K best ---------------------------------------------------------------------------------------
// key: value (order-preserving bits) above the complement of the index: larger key = larger value, ties = lower index
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);          // -0 counts as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ uint64_t make_key(float v, int idx) {
    return ((uint64_t)order_bits(v) << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

struct Best {
    uint64_t* buf;     // this wavefront's LP_CAP entries in LDS
    int count;         // wave-uniform
    float thr;         // no candidate below it is wanted
    uint64_t thr_key;

    __device__ __forceinline__ void init(uint64_t* b) {
        buf = b;
        count = 0;
        thr = LP_LOWEST;                                   // -inf is never a candidate
        thr_key = 0;
    }
    // lower bound of the K-th best from one value per lane (the lanes' maxima)
    __device__ __forceinline__ void bound(float v, int K) {
        const uint32_t o = v == v ? order_bits(v) : 0u;    // a lane with nothing but NaN bounds nothing
        uint32_t t = 0;
#pragma unroll 1
        for (int b = 31; b >= 0; --b) {
            const uint32_t c = t | (1u << b);
            if (__popcll(__ballot(o >= c)) >= K) t = c;
        }
        const float f = order_value(t);
        if (f > thr) thr = f;                              // t = 0 (fewer than K lanes): NaN, no bound
    }
    // keep the K largest of the list; the smallest of them is the new threshold
    __device__ __forceinline__ void cut(int K) {
        wave_sync_lds();
        const int lane = threadIdx.x & 63;
        uint64_t k[LP_CAP / 64];
#pragma unroll
        for (int j = 0; j < LP_CAP / 64; ++j) k[j] = j * 64 + lane < count ? buf[j * 64 + lane] : 0ull;
        wave_sync_lds();
        if (count <= K) return;
        uint64_t t = 0;
#pragma unroll 1
        for (int b = 63; b >= 0; --b) {
            const uint64_t c = t | (1ull << b);
            int n = 0;
#pragma unroll
            for (int j = 0; j < LP_CAP / 64; ++j) n += __popcll(__ballot(k[j] >= c));
            if (n >= K) t = c;
        }
        int n = 0;
#pragma unroll
        for (int j = 0; j < LP_CAP / 64; ++j) {
            const bool keep = k[j] >= t;
            const uint64_t mask = __ballot(keep);
            if (keep) buf[n + lanes_below(mask)] = k[j];
            n += __popcll(mask);
        }
        count = n;
        thr_key = t;
        const float f = order_value((uint32_t)(t >> 32));
        if (f > thr) thr = f;
        wave_sync_lds();
    }
    __device__ __forceinline__ void add(bool want, uint64_t key, int K) {
        uint64_t mask = __ballot(want && key > thr_key);
        if (mask == 0) return;
        if (count + __popcll(mask) > LP_CAP) {
            cut(K);
            mask = __ballot(want && key > thr_key);
        }
        if (want && key > thr_key) buf[count + lanes_below(mask)] = key;
        count += __popcll(mask);
    }
    // at most 64 keys, one per lane (0: none), and each key's rank among them
    __device__ __forceinline__ uint64_t ranked(int K, int& rank) {
        if (count > 64) cut(K);
        wave_sync_lds();
        const int lane = threadIdx.x & 63;
        const uint64_t key = lane < count ? buf[lane] : 0ull;
        rank = 0;
        for (int j = 0; j < count; ++j) {
            const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), j) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, j);
            rank += o > key ? 1 : 0;
        }
        if (lane >= count) rank = 1 << 20;
        wave_sync_lds();
        return key;
    }
};

// ---- one wavefront's share of a row ------------------------------------------------------------------------------------
// Elements [lo, hi) of the row at p, in 16-byte pieces on the address grid (the row may start off it: odd V); `waves`
// wavefronts take turns of 64 pieces, this one is number `wave`.
template <class T, bool TOP>
__device__ __forceinline__ Stat scan_row(const T* p, int lo, int hi, int wave, int waves, Best& best, int K) {
    constexpr int V = 16 / (int)sizeof(T), U = 4;
    const int lane = threadIdx.x & 63;
    const int a = (int)(((uintptr_t)p & 15) / sizeof(T));           // elements between the grid and the row's start
    const int64_t w_lo = ((int64_t)lo + a) / V, w_hi = ((int64_t)hi + a + V - 1) / V;
    Stat st = {LP_LOWEST, 0.0f, 0.0f};
    bool first = true;
    for (int64_t base = w_lo + wave * 64; base < w_hi; base += (int64_t)waves * 64 * U) {
        float x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t e = (base + (int64_t)u * waves * 64 + lane) * V - a;
            if (e >= lo && e + V <= hi) {
                load_f32<T, V>(x[u], p + e);
            } else {
#pragma unroll
                for (int q = 0; q < V; ++q) x[u][q] = (e + q >= lo && e + q < hi) ? (float)p[e + q] : -__builtin_inff();
            }
        }
        float mv = x[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) mv = fmaxf(mv, x[u][q]);
        const float m = fmaxf(st.m, mv), d0 = st.m - m, f = lp_exp(d0);
        float z = 0.0f, s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (base + (int64_t)u * waves * 64 >= w_hi) break;          // wavefront-uniform: nothing but padding from here on
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const float d = x[u][q] - m, e = lp_exp(d);
                z += e;
                s = fmaf(e, fmaxf(d, LP_FLOOR), s);
            }
        }
        st.s = fmaf(f, fmaf(st.z, fmaxf(d0, LP_FLOOR), st.s), s);
        st.z = fmaf(st.z, f, z);
        st.m = m;
        if constexpr (TOP) {
            if (first) best.bound(mv, K);
            first = false;
            if (__ballot(mv >= best.thr) != 0) {
                // one bit per element, then each lane's candidates in turn, read again: the list's code stands here once
                // (once per element it would not fit the instruction cache)
                uint32_t want = 0;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int q = 0; q < V; ++q) want |= x[u][q] >= best.thr ? 1u << (u * V + q) : 0u;
#pragma unroll 1
                while (__ballot(want != 0) != 0) {
                    const int at = want != 0 ? __ffs((int)want) - 1 : 0;
                    const int64_t e = (base + (int64_t)(at / V) * waves * 64 + lane) * V - a + at % V;
                    const float v = want != 0 ? (float)p[e] : -__builtin_inff();
                    best.add(v >= best.thr, make_key(v, (int)e), K);
                    want &= want - 1;
                }
            }
        }
    }
    return st;
}

// ---- what a finished row writes ------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t lp_target(const LogpArgs& a, int64_t row, int t) {
    return a.id64 ? ((const int64_t*)a.tgt)[row * a.T + t] : (int64_t)((const int32_t*)a.tgt)[row * a.T + t];
}
template <class T>
__device__ __forceinline__ void write_stats(const LogpArgs& a, int64_t row, const Stat& st, int lane) {
    const bool none = st.z == 0.0f;                        // every logit is -inf
    const float m = none ? -__builtin_inff() : st.m, lz = none ? 0.0f : logf(st.z);
    if (lane == 0) {
        a.lse[2 * row] = m;
        a.lse[2 * row + 1] = lz;
        a.ent[row] = none ? 0.0f : lz - st.s / st.z;
    }
    if (lane < a.T) {
        const int64_t t = lp_target(a, row, lane);
        float v = 0.0f;                                    // no such item: 0
        if (t >= 0 && t < a.V) v = none ? -__builtin_inff() : ((float)((const T*)a.x)[row * a.ld + t] - m) - lz;
        a.logp[row * a.T + lane] = v;
    }
}
// rank < K: key's place in the list; the places behind the last key are -1 / -inf
__device__ __forceinline__ void write_best(const LogpArgs& a, int64_t row, const Stat& st, uint64_t key, int rank, int found) {
    const int lane = threadIdx.x & 63;
    const float lz = logf(st.z);
    if (rank < a.K) {
        a.top_idx[row * a.K + rank] = (int32_t)~(uint32_t)key;
        a.top_logp[row * a.K + rank] = (order_value((uint32_t)(key >> 32)) - st.m) - lz;
    }
    if (lane >= found && lane < a.K) {
        a.top_idx[row * a.K + lane] = -1;
        a.top_logp[row * a.K + lane] = -__builtin_inff();
    }
}

// the four wavefronts' lists -> the row's K best (called by all 256 threads)
__device__ __forceinline__ void block_best(const LogpArgs& a, int64_t row, const Stat& st, Best& best, uint64_t* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (best.count > 64) best.cut(a.K);
    if (lane >= best.count) best.buf[lane] = 0ull;
    __syncthreads();
    if (wave != 0) return;
    // at most 64 keys of each list: they fit the first wavefront's 256 entries, which its own list begins
#pragma unroll 1
    for (int j = 1; j < 4; ++j) {
        const uint64_t k = all[j * LP_CAP + lane];
        best.add(k != 0, k, a.K);
    }
    int rank;
    const uint64_t mine = best.ranked(a.K, rank);
    write_best(a, row, st, mine, rank, best.count);
}

template <class T, bool TOP>
__global__ __launch_bounds__(256) void logp_row_wave_kernel(LogpArgs a) {
    __shared__ uint64_t buf[TOP ? 4 * LP_CAP : 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.N) return;                                // no workgroup barrier below
    Best best;
    best.init(buf + (TOP ? wave * LP_CAP : 0));
    const Stat st = stat_wave(scan_row<T, TOP>((const T*)a.x + row * a.ld, 0, a.V, 0, 1, best, a.K));
    write_stats<T>(a, row, st, lane);
    if constexpr (TOP) {
        int rank;
        const uint64_t key = best.ranked(a.K, rank);
        write_best(a, row, st, key, rank, best.count);
    }
}

template <class T, bool TOP>
__global__ __launch_bounds__(256) void logp_row_kernel(LogpArgs a) {
    __shared__ uint64_t buf[TOP ? 4 * LP_CAP : 1];
    __shared__ Stat sts[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x / a.splits;
    const int sp = (int)(blockIdx.x % a.splits);
    const int64_t lo = (int64_t)sp * a.seg, hi = lo + a.seg < a.V ? lo + a.seg : a.V;
    Best best;
    best.init(buf + (TOP ? wave * LP_CAP : 0));
    Stat st = stat_wave(scan_row<T, TOP>((const T*)a.x + row * a.ld, (int)lo, (int)hi, wave, 4, best, a.K));
    if (lane == 0) sts[wave] = st;
    if constexpr (TOP) {
        if (a.splits > 1) {
            int rank;
            const uint64_t key = best.ranked(a.K, rank);
            uint64_t* out = a.pkey + (((int64_t)row * a.splits + sp) * 4 + wave) * a.K;
            if (rank < a.K) out[rank] = key;
            if (lane >= best.count && lane < a.K) out[lane] = 0ull;
        }
    }
    __syncthreads();
    st = stat_join(stat_join(sts[0], sts[1]), stat_join(sts[2], sts[3]));
    if (a.splits > 1) {
        if (threadIdx.x == 0) {
            float* o = a.pst + ((int64_t)row * a.splits + sp) * 4;
            o[0] = st.m;
            o[1] = st.z;
            o[2] = st.s;
        }
        return;
    }
    if (wave == 3) write_stats<T>(a, row, st, lane);
    if constexpr (TOP) block_best(a, row, st, best, buf);
}

// joins the parts of a split row: at most 256 statistics, splits * 4 * K keys
template <class T, bool TOP>
__global__ __launch_bounds__(256) void logp_join_kernel(LogpArgs a) {
    __shared__ uint64_t buf[TOP ? 4 * LP_CAP : 1];
    __shared__ Stat sts[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x;
    Stat st = {LP_LOWEST, 0.0f, 0.0f};
    if ((int)threadIdx.x < a.splits) {
        const float* o = a.pst + ((int64_t)row * a.splits + threadIdx.x) * 4;
        st.m = o[0];
        st.z = o[1];
        st.s = o[2];
    }
    st = stat_wave(st);
    if (lane == 0) sts[wave] = st;
    Best best;
    best.init(buf + (TOP ? wave * LP_CAP : 0));
    if constexpr (TOP) {
        const int n = a.splits * 4 * a.K;
        const uint64_t* keys = a.pkey + (int64_t)row * n;
        constexpr int J = 4;                                   // keys a lane requests together (the selection below names them)
        for (int i0 = wave * 64 * J; i0 < n; i0 += 256 * J) {
            uint64_t k[J], top = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int i = i0 + j * 64 + lane;
                k[j] = keys[i < n ? i : n - 1];
                if (i >= n) k[j] = 0;
            }
#pragma unroll
            for (int j = 0; j < J; ++j) top = k[j] > top ? k[j] : top;
            // the K-th best of the lanes' best bounds the K-th best of all: hardly more than K candidates remain
            if (i0 < 256 * J) best.bound(top ? order_value((uint32_t)(top >> 32)) : -__builtin_inff(), a.K);
            uint32_t want = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) want |= k[j] != 0 && order_value((uint32_t)(k[j] >> 32)) >= best.thr ? 1u << j : 0u;
#pragma unroll 1
            while (__ballot(want != 0) != 0) {
                const uint64_t key = want & 1u ? k[0] : want & 2u ? k[1] : want & 4u ? k[2] : k[3];
                best.add(want != 0, key, a.K);
                want &= want - 1;
            }
        }
    }
    __syncthreads();
    st = stat_join(stat_join(sts[0], sts[1]), stat_join(sts[2], sts[3]));
    if (wave == 3) write_stats<T>(a, row, st, lane);
    if constexpr (TOP) block_best(a, row, st, best, buf);
}

// ---- gradient --------------------------------------------------------------------------------------------------------------
struct LogpGradArgs {
    const void* x;
    int64_t ld, N;
    int V;
    const void* tgt;
    int id64, T;
    const float *lse, *ent, *g, *gh;   // g [N, T] or NULL, gh [N] or NULL
    int splits, seg;
    void* dx;                          // [N, V]
};

// ROWS rows (or row parts) per workgroup: 4 = a wavefront each, 1 = all four on one
template <class T, int ROWS>
__global__ __launch_bounds__(256) void logp_grad_kernel(LogpGradArgs a) {
    constexpr int V = 16 / (int)sizeof(T), U = 4, NT = 256 / ROWS;
    const int64_t part = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT, row = part / a.splits;
    const int tid = threadIdx.x % NT;
    if (row >= a.N) return;                                 // whole wavefronts; ROWS = 1: never
    const int64_t lo = part % a.splits * a.seg, hi = lo + a.seg < a.V ? lo + a.seg : a.V;
    const T* p = (const T*)a.x + row * a.ld;
    T* o = (T*)a.dx + row * a.V;
    const float m = a.lse[2 * row], lz = a.lse[2 * row + 1];
    auto target = [&](int t) -> int64_t {
        return a.id64 ? ((const int64_t*)a.tgt)[row * a.T + t] : (int64_t)((const int32_t*)a.tgt)[row * a.T + t];
    };
    float G = 0.0f;
    for (int t = 0; t < a.T; ++t) {
        const int64_t v = target(t);
        G += (v >= 0 && v < a.V) ? a.g[row * a.T + t] : 0.0f;
    }
    const float gh = a.gh ? a.gh[row] : 0.0f, H = a.gh ? a.ent[row] : 0.0f;
    const bool none = m == -__builtin_inff();               // every logit is -inf: no probabilities, no gradient
    auto grad = [&](float x) -> float {
        const float lp = (x - m) - lz, pr = lp_exp(lp);
        return none ? 0.0f : -pr * fmaf(gh, fmaxf(lp, LP_FLOOR) + H, G);
    };
    const int off = (int)(((uintptr_t)p & 15) / sizeof(T));
    if (off == (int)(((uintptr_t)o & 15) / sizeof(T))) {
        const int64_t w_lo = (lo + off) / V, w_hi = (hi + off + V - 1) / V;
        for (int64_t base = w_lo + tid; base < w_hi; base += NT * U) {
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t e = (base + u * NT) * V - off;
                if (e >= lo && e + V <= hi) {
                    load_f32<T, V>(x[u], p + e);
                } else {
#pragma unroll
                    for (int q = 0; q < V; ++q) x[u][q] = (e + q >= lo && e + q < hi) ? (float)p[e + q] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t e = (base + u * NT) * V - off;
                if (e >= hi) break;
#pragma unroll
                for (int q = 0; q < V; ++q) x[u][q] = grad(x[u][q]);
                if (e >= lo && e + V <= hi) {
                    store_f32<T, V>(o + e, x[u]);
                } else {
#pragma unroll
                    for (int q = 0; q < V; ++q)
                        if (e + q >= lo && e + q < hi) o[e + q] = (T)x[u][q];
                }
            }
        }
    } else {
        // rows of x and dx lie differently on the 16-byte grid, as where the logits are a view without one item: an element at
        // a time (4096 x 30000 bf16 228 us, 105 from rows that lie alike; 4096 x 3707 fp16 25.9 and 17.5)
#pragma unroll 8
        for (int64_t e = lo + tid; e < hi; e += NT) o[e] = (T)grad((float)p[e]);
    }
    if (a.T == 0) return;
    // the targets' own terms: added before the one rounding, so their elements are written again, by the first of the
    // entries that name the item (its repeats are summed in list order) -- after the first writes have arrived
    if constexpr (ROWS == 1) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
    if (tid < a.T && !none) {
        const int64_t v = target(tid);
        if (v >= lo && v < hi) {
            float s = 0.0f;
            bool mine = true;
            for (int q = 0; q < a.T; ++q)
                if (target(q) == v) {
                    if (q < tid) mine = false;
                    s += a.g[row * a.T + q];
                }
            if (mine) o[v] = (T)(grad((float)p[v]) + s);
        }
    }
}

// workgroups per row and elements each: enough of them to fill the chip, none below 4096 elements (8 x 100001 bf16, K = 10:
// 15.6 us; 17.0 us with a limit of 2048, 18.4 us with 16384; 128 x 50000: 17.0 us, 19.9 us with a limit of 16384)
static void logp_split(int64_t N, int V, int64_t want, int* splits, int* seg) {
    int64_t s = (want + N - 1) / N;
    if (s > V / 4096) s = V / 4096;
    if (s > LP_MAX_SPLITS) s = LP_MAX_SPLITS;
    if (s < 1) s = 1;
    const int64_t e = align_up((V + s - 1) / s, 1024);
    *seg = (int)(e < V ? e : V);
    *splits = (int)(((int64_t)V + *seg - 1) / *seg);
}
constexpr int64_t LP_FILL = 1024;      // 4 workgroups per CU
static bool logp_wave_rows(int64_t N, int64_t V) { return V <= 2048 || (V <= 16384 && N >= 2048); }

}  // namespace dr

extern "C" int64_t dr_item_logprobs_bytes(int64_t N, int64_t V, int32_t K) {
    using namespace dr;
    if (N < 0 || V < 1 || V > 0x7FFFFFFF || K < 0 || K > LP_MAX_K) return DR_ERR_ARG;
    if (N == 0 || logp_wave_rows(N, V)) return 0;
    int splits, seg;
    logp_split(N, (int)V, LP_FILL, &splits, &seg);
    if (splits == 1) return 0;
    return align_up(N * splits * 16, 256) + align_up(N * splits * 4 * (int64_t)K * 8, 256);
}

extern "C" int32_t dr_item_logprobs_forward(const void* logits, int64_t N, int64_t V, int64_t ld, int32_t dtype,
                                            const void* targets, int32_t id_bits, int32_t T, int32_t K, float* logp,
                                            float* entropy, float* lse, int32_t* top_idx, float* top_logp, void* ws,
                                            int64_t ws_bytes, void* stream) {
    using namespace dr;
    DR_REQUIRE(dtype_ok(dtype), "dr_item_logprobs_forward: dtype %d", dtype);
    DR_REQUIRE(N >= 0 && V >= 1 && V <= 0x7FFFFFFF && ld >= V, "dr_item_logprobs_forward: bad sizes (N=%lld V=%lld ld=%lld)",
               (long long)N, (long long)V, (long long)ld);
    DR_REQUIRE(T >= 0 && T <= LP_MAX_T && K >= 0 && K <= LP_MAX_K, "dr_item_logprobs_forward: T=%d or K=%d beyond %d", T, K,
               LP_MAX_K);
    DR_REQUIRE(T == 0 || id_bits == 32 || id_bits == 64, "dr_item_logprobs_forward: id_bits must be 32 or 64");
    if (N == 0) return DR_OK;
    DR_REQUIRE(logits && entropy && lse && (T == 0 || (targets && logp)) && (K == 0 || (top_idx && top_logp)),
               "dr_item_logprobs_forward: NULL pointer");
    DR_REQUIRE(aligned_to(logits, dtype_size(dtype)), "dr_item_logprobs_forward: logits not aligned to the element size");
    const int64_t need = dr_item_logprobs_bytes(N, V, K);
    DR_REQUIRE(need == 0 || ws != nullptr, "dr_item_logprobs_forward: workspace is NULL");
    DR_REQUIRE(aligned_to(ws, 256), "dr_item_logprobs_forward: workspace is not 256-byte aligned");
    if (ws_bytes < need)
        DR_FAIL(DR_ERR_WORKSPACE, "dr_item_logprobs_forward: workspace %lld < required %lld", (long long)ws_bytes, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    LogpArgs a;
    a.x = logits;
    a.ld = ld;
    a.N = N;
    a.V = (int)V;
    a.tgt = targets;
    a.id64 = id_bits == 64;
    a.T = T;
    a.K = K;
    a.logp = logp;
    a.ent = entropy;
    a.lse = lse;
    a.top_idx = top_idx;
    a.top_logp = top_logp;
    a.splits = 1;
    a.seg = a.V;
    a.pst = nullptr;
    a.pkey = nullptr;
    if (logp_wave_rows(N, V)) {
        DR_REQUIRE((N + 3) / 4 < LP_MAX_GRID, "dr_item_logprobs_forward: too many rows");
#define LP_WAVE(T_)                                                                                                     \
    if (K)                                                                                                              \
        DR_LAUNCH_NAMED("logp_row_wave_kernel", (logp_row_wave_kernel<T_, true>), dim3((unsigned)((N + 3) / 4)),        \
                        dim3(256), 0, st, a);                                                                           \
    else                                                                                                                \
        DR_LAUNCH_NAMED("logp_row_wave_kernel", (logp_row_wave_kernel<T_, false>), dim3((unsigned)((N + 3) / 4)),       \
                        dim3(256), 0, st, a)
        DR_BY_DTYPE(dtype, LP_WAVE);
#undef LP_WAVE
        DR_CHECK_LAUNCH("logp_row_wave_kernel");
        return DR_OK;
    }
    logp_split(N, a.V, LP_FILL, &a.splits, &a.seg);
    DR_REQUIRE(N * a.splits < LP_MAX_GRID, "dr_item_logprobs_forward: too many rows");
    if (a.splits > 1) {
        a.pst = (float*)ws;
        a.pkey = (uint64_t*)((char*)ws + align_up(N * a.splits * 16, 256));
    }
    const unsigned grid = (unsigned)(N * a.splits);
#define LP_ROW(T_)                                                                                                      \
    if (K)                                                                                                              \
        DR_LAUNCH_NAMED("logp_row_kernel", (logp_row_kernel<T_, true>), dim3(grid), dim3(256), 0, st, a);               \
    else                                                                                                                \
        DR_LAUNCH_NAMED("logp_row_kernel", (logp_row_kernel<T_, false>), dim3(grid), dim3(256), 0, st, a)
    DR_BY_DTYPE(dtype, LP_ROW);
#undef LP_ROW
    DR_CHECK_LAUNCH("logp_row_kernel");
    if (a.splits > 1) {
#define LP_JOIN(T_)                                                                                                     \
    if (K)                                                                                                              \
        DR_LAUNCH_NAMED("logp_join_kernel", (logp_join_kernel<T_, true>), dim3((unsigned)N), dim3(256), 0, st, a);      \
    else                                                                                                                \
        DR_LAUNCH_NAMED("logp_join_kernel", (logp_join_kernel<T_, false>), dim3((unsigned)N), dim3(256), 0, st, a)
        DR_BY_DTYPE(dtype, LP_JOIN);
#undef LP_JOIN
        DR_CHECK_LAUNCH("logp_join_kernel");
    }
    return DR_OK;
}

extern "C" int32_t dr_item_logprobs_backward(const void* logits, int64_t N, int64_t V, int64_t ld, int32_t dtype,
                                             const void* targets, int32_t id_bits, int32_t T, const float* lse,
                                             const float* entropy, const float* g_logp, const float* g_entropy,
                                             void* glogits, void* stream) {
    using namespace dr;
    DR_REQUIRE(dtype_ok(dtype), "dr_item_logprobs_backward: dtype %d", dtype);
    DR_REQUIRE(N >= 0 && V >= 1 && V <= 0x7FFFFFFF && ld >= V, "dr_item_logprobs_backward: bad sizes (N=%lld V=%lld ld=%lld)",
               (long long)N, (long long)V, (long long)ld);
    DR_REQUIRE(T >= 0 && T <= LP_MAX_T, "dr_item_logprobs_backward: T=%d beyond %d", T, LP_MAX_T);
    DR_REQUIRE(T == 0 || id_bits == 32 || id_bits == 64, "dr_item_logprobs_backward: id_bits must be 32 or 64");
    if (N == 0) return DR_OK;
    DR_REQUIRE(logits && lse && glogits && (T == 0 || (targets && g_logp)) && (!g_entropy || entropy),
               "dr_item_logprobs_backward: NULL pointer");
    DR_REQUIRE(aligned_to(logits, dtype_size(dtype)) && aligned_to(glogits, dtype_size(dtype)),
               "dr_item_logprobs_backward: a pointer is not aligned to its element size");
    LogpGradArgs a;
    a.x = logits;
    a.ld = ld;
    a.N = N;
    a.V = (int)V;
    a.tgt = targets;
    a.id64 = id_bits == 64;
    a.T = T;
    a.lse = lse;
    a.ent = entropy;
    a.g = g_logp;
    a.gh = g_entropy;
    a.dx = glogits;
    hipStream_t st = (hipStream_t)stream;
    if (logp_wave_rows(N, V)) {
        a.splits = 1;
        a.seg = a.V;
        DR_REQUIRE((N + 3) / 4 < LP_MAX_GRID, "dr_item_logprobs_backward: too many rows");
#define LP_GRAD(T_) \
    DR_LAUNCH_NAMED("logp_grad_kernel", (logp_grad_kernel<T_, 4>), dim3((unsigned)((N + 3) / 4)), dim3(256), 0, st, a)
        DR_BY_DTYPE(dtype, LP_GRAD);
#undef LP_GRAD
    } else {
        logp_split(N, a.V, LP_FILL, &a.splits, &a.seg);
        DR_REQUIRE(N * a.splits < LP_MAX_GRID, "dr_item_logprobs_backward: too many rows");
#define LP_GRAD(T_) \
    DR_LAUNCH_NAMED("logp_grad_kernel", (logp_grad_kernel<T_, 1>), dim3((unsigned)(N * a.splits)), dim3(256), 0, st, a)
        DR_BY_DTYPE(dtype, LP_GRAD);
#undef LP_GRAD
    }
    DR_CHECK_LAUNCH("logp_grad_kernel");
    return DR_OK;
}
