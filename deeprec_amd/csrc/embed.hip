// Embedding lookup with scaling, fp32 / fp16 / bf16 tables, and its gradient by sorted ids.
//   forward   out[e, :] = scale * table[ids[e], :]            (an id outside [0, rows): a zero row, as dr_gather_f32)
//   backward  grad[r, :] = scale * sum over e with ids[e] == r of gout[e, :]   for EVERY row r (untouched rows: 0);
//             ids equal to padding, or outside [0, rows), contribute nothing.
// HBM-bound both ways.  Sums are fp32 in a fixed order (sorted list cut into chunks of 8 or 32 entries, entries in list
// order inside a chunk, a row's chunks in ascending order): the same ids and gradients give the same bits, with no atomics.
#include <utility>

#include "dr_lsd_sort.h"
#include "dr_types.h"

namespace dr {

constexpr int EMB_MAX_D = 32768;
// Sorted entries a group of lanes sums: few where the list is short and the chip would idle (whole gradient of 20000 rows of
// 128 bf16: 29 us with 8, 33 us with 32; of 100000: 41 and 37 us)
static int embed_chunk(int64_t n) { return n <= 65536 ? 8 : 32; }

// ---- forward -------------------------------------------------------------------------------------------------------
// A block owns R whole rows = R * cpr vectors of V elements, dealt to its threads in order, so every lane moves 16 bytes
// (or the widest piece the row size and the bases allow) whatever d is; U independent id -> row chains per thread.
// 204800 rows of 128 bf16 out of 100001: 15 us = 5.3 TB/s of rows written and distinct rows read; 5000 x 150 fp32: 3.8 us.
template <class T, class Id, int V>
__global__ __launch_bounds__(256) void embed_forward_kernel(const T* __restrict__ table, int64_t rows, int d, int cpr,
                                                            uint64_t magic, const Id* __restrict__ ids, int64_t n, int R,
                                                            float scale, T* __restrict__ out) {
    constexpr int U = 4;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < n; r0 += (int64_t)gridDim.x * R) {
        const int nr = (int)(n - r0 < R ? n - r0 : R), total = nr * cpr;
        for (int base = threadIdx.x; base < total; base += 256 * U) {
            int64_t id[U];
            int c[U];
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = base + u * 256 < total ? base + u * 256 : total - 1;
                const int r = (int)(((uint64_t)(uint32_t)w * magic) >> 32);   // w / cpr: exact, as w, cpr < 65536
                c[u] = w - r * cpr;
                id[u] = (int64_t)ids[r0 + r];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool ok = id[u] >= 0 && id[u] < rows;
                load_f32<T, V>(v[u], table + (ok ? id[u] : 0) * d + c[u] * V);
#pragma unroll
                for (int x = 0; x < V; ++x) v[u][x] = ok ? v[u][x] * scale : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = base + u * 256;
                if (w < total) store_f32<T, V>(out + r0 * d + (int64_t)w * V, v[u]);
            }
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// Stable sort of (id, list position), then the sums.  At 2 x 10^5 ids the sort is launches and latency, not bytes, so it
// takes the fewest passes that cover the table's rows (digits of 8 to 11 bits: 2 passes up to 2^22 rows), and while it
// runs most of the chip would idle: its launches carry extra workgroups that clear the gradient table (rows no id names
// stay 0), which therefore costs next to nothing.
constexpr int SRT_T = 512, SRT_WAVES = SRT_T / 64, SRT_IPT = 4, SRT_TILE = SRT_T * SRT_IPT;
// beyond, every workgroup would read too many tile histograms: lsd_sort (gradient of 400000 rows of 64 fp32: 69 us, 93 us with
// lsd_sort)
constexpr int SRT_MAX_TILES = 512;
constexpr int64_t SRT_MAX_N = SRT_MAX_TILES * SRT_TILE;
// up to here a workgroup counts all keys itself instead of a histogram launch (gradient of 8192 rows of 64 fp32: 22.6 us, 26.5 us
// with the launch; of 16000: 33.4 and 28.5 us)
constexpr int SRT_DIRECT_TILES = 4;

template <class Id>
struct EmbedKeys {  // ids -> sort keys; ids that contribute nothing sort behind every row
    const Id* ids;
    int64_t rows, padding;
    __device__ __forceinline__ uint32_t key(int64_t e) const {
        const int64_t id = (int64_t)ids[e];
        return (id < 0 || id >= rows || id == padding) ? (uint32_t)rows : (uint32_t)id;
    }
    __device__ __forceinline__ int32_t val(int64_t e) const { return (int32_t)e; }
};

struct EmbedPairs {  // a previous pass's output
    const uint2* pairs;
    __device__ __forceinline__ uint32_t key(int64_t e) const { return pairs[e].x; }
    __device__ __forceinline__ int32_t val(int64_t e) const { return (int32_t)pairs[e].y; }
};

// `count` 16-byte pieces of zeros from `base` on, written by workgroups first, first + 1, .. first + blocks - 1
struct EmbedFill {
    uint4* base;
    int64_t count;
    int first, blocks;
};
__device__ __forceinline__ void embed_fill(const EmbedFill& f, int block) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 z = {0, 0, 0, 0};
    const int64_t per = (f.count + f.blocks - 1) / f.blocks, lo = block * per, hi = lo + per < f.count ? lo + per : f.count;
#pragma unroll 4
    for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) reinterpret_cast<u32x4*>(f.base)[i] = z;
}
template <class T>
__global__ __launch_bounds__(256) void embed_zero_kernel(EmbedFill f, T* __restrict__ tail, int n_tail) {
    embed_fill(f, (int)blockIdx.x);
    if (blockIdx.x == 0 && (int)threadIdx.x < n_tail) tail[threadIdx.x] = (T)0.0f;
}

// digit counts of every tile
template <int BITS, class Src>
__global__ __launch_bounds__(SRT_T) void embed_hist_kernel(Src src, int n, unsigned shift, uint16_t* __restrict__ hist,
                                                           EmbedFill fill) {
    constexpr int BINS = 1 << BITS;
    __shared__ int bins[BINS];
    if ((int)blockIdx.x >= fill.first) {
        embed_fill(fill, (int)blockIdx.x - fill.first);
        return;
    }
    const int base = (int)blockIdx.x * SRT_TILE + (int)threadIdx.x;
    uint32_t key[SRT_IPT];
#pragma unroll
    for (int q = 0; q < SRT_IPT; ++q) key[q] = src.key(base + q * SRT_T < n ? base + q * SRT_T : n - 1);
    for (int d = threadIdx.x; d < BINS; d += SRT_T) bins[d] = 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < SRT_IPT; ++q)
        if (base + q * SRT_T < n) atomicAdd(&bins[(key[q] >> shift) & (BINS - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < BINS; d += SRT_T) hist[(int64_t)blockIdx.x * BINS + d] = (uint16_t)bins[d];
}

// exclusive sum of one value per thread over the workgroup
__device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y = __shfl_up(s, off, 64);
        if (lane >= off) s += y;
    }
    if (lane == 63) red[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += red[w];
    __syncthreads();
    return before + s - x;
}

// Places every key of a tile: keys with a smaller digit, equal digits in earlier tiles, equal digits earlier in the tile.
// A wavefront takes 256 consecutive keys in four rounds of 64; lanes with equal digits find each other by one ballot per
// bit, the first of them moves the wavefront's counter of that digit.  No atomics whose order matters.
template <int BITS, class Src>
__global__ __launch_bounds__(SRT_T) void embed_scatter_kernel(Src src, int n, unsigned shift, const uint16_t* __restrict__ hist,
                                                              int ntiles, uint2* __restrict__ out, EmbedFill fill) {
    constexpr int BINS = 1 << BITS, BPT = BINS > SRT_T ? BINS / SRT_T : 1;
    __shared__ uint32_t cnt[SRT_WAVES][BINS];       // a wavefront's keys per digit, then where they go
    __shared__ uint32_t red[SRT_WAVES];
    if ((int)blockIdx.x >= fill.first) {
        embed_fill(fill, (int)blockIdx.x - fill.first);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tile = (int)blockIdx.x;
    // the tile's keys and payloads first: they arrive while the counts are put together
    uint32_t key[SRT_IPT], rank[SRT_IPT];
    int32_t val[SRT_IPT];
    const int k0 = tile * SRT_TILE + wave * (64 * SRT_IPT) + lane;
#pragma unroll
    for (int q = 0; q < SRT_IPT; ++q) {
        const int e = k0 + q * 64 < n ? k0 + q * 64 : n - 1;
        key[q] = src.key(e);
        val[q] = src.val(e);
    }
    // cnt[0]: keys per digit in earlier tiles, cnt[1]: in this one and later ones
    for (int d = tid; d < BINS; d += SRT_T) cnt[0][d] = cnt[1][d] = 0;
    __syncthreads();
    if (hist) {
        // pairs of digits x parts of the tile list over the threads, 32 tiles of a part requested together: the table was
        // written by other XCDs, a round trip to it is what this step costs
        constexpr int PAIRS = BINS / 2, PARTS = PAIRS < SRT_T ? SRT_T / PAIRS : 1;
        const uint32_t* h2 = reinterpret_cast<const uint32_t*>(hist);
        const int per = (ntiles + PARTS - 1) / PARTS, t_lo = tid / PAIRS * per, t_hi = t_lo + per < ntiles ? t_lo + per : ntiles;
        for (int p = tid % PAIRS; p < PAIRS; p += SRT_T) {
            uint32_t e0 = 0, e1 = 0, r0 = 0, r1 = 0;
            for (int t0 = t_lo; t0 < t_hi; t0 += 32) {
                uint32_t h[32];
#pragma unroll
                for (int q = 0; q < 32; ++q) h[q] = h2[(int64_t)(t0 + q < t_hi ? t0 + q : t_lo) * PAIRS + p];
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    const uint32_t v = t0 + q < t_hi ? h[q] : 0u;
                    if (t0 + q < tile) {
                        e0 += v & 0xFFFFu;
                        e1 += v >> 16;
                    } else {
                        r0 += v & 0xFFFFu;
                        r1 += v >> 16;
                    }
                }
            }
            atomicAdd(&cnt[0][2 * p], e0);
            atomicAdd(&cnt[0][2 * p + 1], e1);
            atomicAdd(&cnt[1][2 * p], r0);
            atomicAdd(&cnt[1][2 * p + 1], r1);
        }
    } else {                                                     // few keys: count all of them here
        uint32_t k[SRT_DIRECT_TILES][SRT_IPT];
#pragma unroll
        for (int t = 0; t < SRT_DIRECT_TILES; ++t)
#pragma unroll
            for (int q = 0; q < SRT_IPT; ++q) {
                const int e = t * SRT_TILE + q * SRT_T + tid;
                k[t][q] = src.key(e < n ? e : n - 1);
            }
#pragma unroll
        for (int t = 0; t < SRT_DIRECT_TILES; ++t)
#pragma unroll
            for (int q = 0; q < SRT_IPT; ++q)
                if (t * SRT_TILE + q * SRT_T + tid < n) atomicAdd(&cnt[t < tile ? 0 : 1][(k[t][q] >> shift) & (BINS - 1)], 1u);
    }
    __syncthreads();
    uint32_t tot[BPT], pre[BPT];
    const int d0 = tid * BPT;
    const bool own = d0 < BINS;
#pragma unroll
    for (int x = 0; x < BPT; ++x) {
        pre[x] = own ? cnt[0][d0 + x] : 0u;
        tot[x] = own ? pre[x] + cnt[1][d0 + x] : 0u;
    }
    __syncthreads();
    for (int d = tid; d < BINS * SRT_WAVES; d += SRT_T) (&cnt[0][0])[d] = 0;
    uint32_t mine = 0;
#pragma unroll
    for (int x = 0; x < BPT; ++x) mine += tot[x];
    uint32_t base = block_exclusive(mine, red);                  // its barriers also order the clearing above
    // rank inside the wavefront's 256 keys
#pragma unroll
    for (int q = 0; q < SRT_IPT; ++q) {
        const bool in = k0 + q * 64 < n;
        const uint32_t d = (key[q] >> shift) & (BINS - 1);
        uint64_t same = __ballot(in);
#pragma unroll
        for (int b = 0; b < BITS; ++b) {
            const uint64_t ones = __ballot((d >> b) & 1u);
            same &= (d >> b) & 1u ? ones : ~ones;
        }
        const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0u));
        uint32_t before = 0;
        if (in) before = cnt[wave][d];
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) cnt[wave][d] = before + (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[q] = before + (uint32_t)below;
    }
    __syncthreads();
    if (own) {
#pragma unroll
        for (int x = 0; x < BPT; ++x) {
            uint32_t at = base + pre[x];
#pragma unroll
            for (int w = 0; w < SRT_WAVES; ++w) {
                const uint32_t c = cnt[w][d0 + x];
                cnt[w][d0 + x] = at;
                at += c;
            }
            base += tot[x];
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < SRT_IPT; ++q) {
        if (k0 + q * 64 < n) {
            const uint32_t pos = cnt[wave][(key[q] >> shift) & (BINS - 1)] + rank[q];
            out[pos] = make_uint2(key[q], (uint32_t)val[q]);   // one scattered write of 8 bytes, not two of 4
        }
    }
}

struct EmbedArgs {
    const uint32_t* keys;   // sorted keys (every step-th word); those >= rows contribute nothing and stand last
    const uint32_t* spos;   // their list positions, likewise
    int step;
    int64_t n, rows, chunks;
    int chunk, d;
    float scale;
    float* part;            // [chunks, 2, d] sums of the runs that cross a chunk border: first run, last run
    uint8_t* state;         // [chunks] RUN_*
};
constexpr uint8_t RUN_BEGINS = 1;   // the last run of the chunk begins in it and goes on behind it
constexpr uint8_t RUN_FILLS = 2;    // one run fills the chunk and goes on on both sides

// One group of LPR lanes per chunk.  A run (equal keys) that lies inside the chunk is finished here; the part of a run that
// began in an earlier chunk goes to part[chunk][0], the part of one that goes on behind the chunk to part[chunk][1] (a run
// that does both: [0]).  The chunk's keys and positions are fetched once, spread over the lanes, so that the only
// dependent step left is position -> row, up to 16 rows in flight.  204800 entries of 128 bf16: 16.6 us = 3.2 TB/s (joins 8 us);
// 3668 entries of 95 fp32: 4.2 us.
template <class T, int V, int LPR, int CH>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedArgs a, const T* __restrict__ gout, T* __restrict__ grad) {
    constexpr int E = CH / LPR > 0 ? CH / LPR : 1;                  // entries a lane keeps
    constexpr int DEPTH = CH < 16 ? CH : 16;                        // gradient rows in flight
    const int64_t chunk = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
    const int lane = threadIdx.x % LPR, group0 = (threadIdx.x & 63) - lane;
    if (chunk >= a.chunks) return;                                  // whole groups leave
    const int64_t s0 = chunk * CH;
    const int m = (int)(a.n - s0 < CH ? a.n - s0 : CH);
    uint32_t keys[E];
    uint32_t spos[E];
#pragma unroll
    for (int x = 0; x < E; ++x) {
        const int q = x * LPR + lane;
        const int64_t s = s0 + (q < m ? q : m - 1);
        keys[x] = a.keys[s * a.step];
        spos[x] = a.spos[s * a.step];
    }
    const uint32_t rows = (uint32_t)a.rows, none = 0xFFFFFFFFu;
    const uint32_t before = s0 > 0 ? a.keys[(s0 - 1) * a.step] : none, behind = s0 + m < a.n ? a.keys[(s0 + m) * a.step] : none;
    auto entry = [&](const auto (&r)[E], int q) { return __shfl(r[q / LPR < E ? q / LPR : 0], group0 + q % LPR, 64); };
    const uint32_t k_first = entry(keys, 0), k_last = __shfl(keys[(m - 1) / LPR < E ? (m - 1) / LPR : 0], group0 + (m - 1) % LPR, 64);
    if (lane == 0 && blockIdx.y == 0) {
        uint8_t st = 0;
        if (k_last < rows && k_last == behind) st = k_first == k_last && before == k_first ? RUN_FILLS : RUN_BEGINS;
        a.state[chunk] = st;
    }
    if (k_first >= rows) return;                                    // sorted: nothing from here on contributes
    const int c = (int)blockIdx.y * LPR * V + lane * V;             // this workgroup's columns
    const bool on = c < a.d;                                        // every lane of the group stays for the shuffles
    float acc[V];
#pragma unroll
    for (int x = 0; x < V; ++x) acc[x] = 0.0f;
    uint32_t run = k_first;
    bool carried = before == k_first;
    auto flush = [&](uint32_t next) {                           // the run ends; `next`: the key behind it
        if (!on) return;
        if (carried) {
            store_f32<float, V>(a.part + (chunk * 2) * a.d + c, acc);
        } else if (next == run) {
            store_f32<float, V>(a.part + (chunk * 2 + 1) * a.d + c, acc);
        } else {
#pragma unroll
            for (int x = 0; x < V; ++x) acc[x] *= a.scale;
            store_f32<T, V>(grad + (int64_t)run * a.d + c, acc);
        }
    };
    const T* col = gout + (on ? c : 0);
#pragma unroll
    for (int q0 = 0; q0 < CH; q0 += DEPTH) {
        // unconditional loads of valid rows (entries behind the list repeat its last): under a condition each would
        // wait for the one before
        typename VecType<T, V>::type v[DEPTH];
        uint32_t key[DEPTH];
#pragma unroll
        for (int q = 0; q < DEPTH; ++q)
            v[q] = *reinterpret_cast<const typename VecType<T, V>::type*>(col + (int64_t)entry(spos, q0 + q) * a.d);
#pragma unroll
        for (int q = 0; q < DEPTH; ++q) key[q] = entry(keys, q0 + q);
#pragma unroll
        for (int q = 0; q < DEPTH; ++q) {
            if (q0 + q >= m || key[q] >= rows) continue;
            if (key[q] != run) {
                flush(key[q]);
                run = key[q];
                carried = false;
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] = 0.0f;
            }
            if constexpr (V == 1) {
                acc[0] += (float)v[q];
            } else {
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] += (float)v[q][x];
            }
        }
    }
    flush(k_last < rows ? behind : none);
}

// Joins the runs that cross chunk borders.  A workgroup looks at four chunks; for each in which such a run begins, it
// follows the chunks' states to the run's end (64 at a time) and adds the parts up: its 256 / LPR lane groups take every
// (256 / LPR)-th chunk, the groups' sums are added in order.
template <class T, int V, int LPR>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedArgs a, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / LPR;
    __shared__ float red[GROUPS][LPR * V];
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, wl = threadIdx.x & 63;
    // the four chunks' states in one load (the array is padded)
    const uint32_t states = reinterpret_cast<const uint32_t*>(a.state)[blockIdx.x];
    for (int j = 0; j < 4; ++j) {
        const int64_t chunk = (int64_t)blockIdx.x * 4 + j;
        if (chunk >= a.chunks || ((states >> (8 * j)) & 255u) != RUN_BEGINS) continue;   // workgroup-uniform
        int64_t last = chunk + 1;                                             // last chunk the run reaches
        for (;;) {
            const int64_t at = last + wl;
            const uint64_t ends = __ballot(at >= a.chunks - 1 || a.state[at < a.chunks ? at : a.chunks - 1] != RUN_FILLS);
            if (ends) {
                last += __ffsll((unsigned long long)ends) - 1;
                break;
            }
            last += 64;
        }
        const int64_t run = (int64_t)a.keys[((chunk + 1) * a.chunk - 1) * a.step];
        const int c = (int)blockIdx.y * LPR * V + lane * V;
        float acc[V];
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] = 0.0f;
        if (c < a.d)
#pragma unroll 8
            for (int64_t q = chunk + group; q <= last; q += GROUPS) {
                float v[V];
                load_f32<float, V>(v, a.part + (q * 2 + (q == chunk ? 1 : 0)) * a.d + c);
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] += v[x];
            }
#pragma unroll
        for (int x = 0; x < V; ++x) red[group][lane * V + x] = acc[x];
        __syncthreads();
        if (group == 0 && c < a.d) {
            const int parts = (int)(last - chunk + 1 < GROUPS ? last - chunk + 1 : GROUPS);
            for (int g = 1; g < parts; ++g)
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] += red[g][lane * V + x];
#pragma unroll
            for (int x = 0; x < V; ++x) acc[x] *= a.scale;
            store_f32<T, V>(grad + run * a.d + c, acc);
        }
        __syncthreads();
    }
}

struct EmbedLayout {
    int64_t pairs_a, pairs_b, hist, state, part, total;
};
// digit width and number of passes that cover keys up to `rows` (the sentinel) with n keys
static void embed_digits(int64_t rows, unsigned* bits, unsigned* passes) {
    unsigned end_bit = 1;
    while (end_bit < 31 && ((uint64_t)rows >> end_bit) != 0) ++end_bit;
    *passes = end_bit <= 11 ? 1 : (end_bit <= 22 ? 2 : 3);
    *bits = (end_bit + *passes - 1) / *passes;
    if (*bits < 8) *bits = 8;
}
static EmbedLayout embed_layout(int64_t n, int d) {
    EmbedLayout L;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = off;
        off += align_up(bytes, 256);
        return o;
    };
    const int64_t chunks = (n + embed_chunk(n) - 1) / embed_chunk(n);
    L.pairs_a = take(n * 8);
    L.pairs_b = take(n * 8);
    L.hist = take(n <= SRT_MAX_N ? (n + SRT_TILE - 1) / SRT_TILE * (1 << 11) * 2 : lsd_scratch_bytes(n));
    L.state = take(chunks);
    L.part = take(chunks * 2 * (int64_t)d * 4);
    L.total = off;
    return L;
}

// widest piece of a row, in elements, that d and the two bases allow (16 bytes at most)
static int embed_width(int dt, int d, const void* p, const void* q) {
    int v = 16 / dtype_size(dt);
    while (v > 1 && (d % v != 0 || !aligned_to(p, v * dtype_size(dt)) || !aligned_to(q, v * dtype_size(dt)))) v >>= 1;
    return v;
}
static uint64_t magic_for(int cpr) { return ((1ull << 32) + cpr - 1) / cpr; }

template <class T, class Id, int V>
static int embed_forward_launch(const void* table, int64_t rows, int d, const void* ids, int64_t n, float scale, void* out,
                                hipStream_t st) {
    const int cpr = d / V;
    // rows per block: up to 2048 pieces (8 per thread), fewer while that leaves less than 4 blocks per CU (20000 rows of 32 bf16:
    // 2.9 us, 3.8 us with 2048 pieces throughout)
    int64_t R = 2048 / cpr;
    if (R > n / 1024) R = n / 1024;
    if (R < 1) R = 1;
    const int64_t blocks = (n + R - 1) / R;
    const int grid = (int)(blocks < (1 << 20) ? blocks : (1 << 20));
    DR_LAUNCH_NAMED("embed_forward_kernel", (embed_forward_kernel<T, Id, V>), dim3(grid), dim3(256), 0, st, (const T*)table,
                    rows, d, cpr, magic_for(cpr), (const Id*)ids, n, (int)R, scale, (T*)out);
    DR_CHECK_LAUNCH("embed_forward_kernel");
    return DR_OK;
}
template <class T, class Id>
static int embed_forward_t(int dt, const void* table, int64_t rows, int d, const void* ids, int64_t n, float scale,
                           void* out, hipStream_t st) {
    switch (embed_width(dt, d, table, out)) {
        case 8:
            if constexpr (sizeof(T) == 2) return embed_forward_launch<T, Id, 8>(table, rows, d, ids, n, scale, out, st);
        case 4: return embed_forward_launch<T, Id, 4>(table, rows, d, ids, n, scale, out, st);
        case 2: return embed_forward_launch<T, Id, 2>(table, rows, d, ids, n, scale, out, st);
        default: return embed_forward_launch<T, Id, 1>(table, rows, d, ids, n, scale, out, st);
    }
}

template <class T, int V, int LPR>
static int embed_sum_launch(const EmbedArgs& a, const void* gout, void* grad, hipStream_t st) {
    const int64_t blocks = (a.chunks * LPR + 255) / 256;
    DR_REQUIRE(blocks < (1ll << 24), "dr_embed_backward: too many blocks");      // a launch counts threads in 32 bits
    const unsigned cols = (unsigned)((a.d + LPR * V - 1) / (LPR * V));      // wide rows: workgroups side by side
    if (a.chunk == 8)
        DR_LAUNCH_NAMED("embed_sum_kernel", (embed_sum_kernel<T, V, LPR, 8>), dim3((unsigned)blocks, cols), dim3(256), 0, st, a,
                        (const T*)gout, (T*)grad);
    else
        DR_LAUNCH_NAMED("embed_sum_kernel", (embed_sum_kernel<T, V, LPR, 32>), dim3((unsigned)blocks, cols), dim3(256), 0, st, a,
                        (const T*)gout, (T*)grad);
    DR_CHECK_LAUNCH("embed_sum_kernel");
    if (a.chunks > 1) {
        DR_LAUNCH_NAMED("embed_join_kernel", (embed_join_kernel<T, V, LPR>), dim3((unsigned)((a.chunks + 3) / 4), cols), dim3(256),
                        0, st, a, (T*)grad);
        DR_CHECK_LAUNCH("embed_join_kernel");
    }
    return DR_OK;
}
template <class T, int V>
static int embed_sum_v(const EmbedArgs& a, const void* gout, void* grad, hipStream_t st) {
    const int cpr = a.d / V;
    if (cpr <= 4) return embed_sum_launch<T, V, 4>(a, gout, grad, st);
    if (cpr <= 8) return embed_sum_launch<T, V, 8>(a, gout, grad, st);
    if (cpr <= 16) return embed_sum_launch<T, V, 16>(a, gout, grad, st);
    if (cpr <= 32) return embed_sum_launch<T, V, 32>(a, gout, grad, st);
    return embed_sum_launch<T, V, 64>(a, gout, grad, st);
}

// the part of the table that launch `step` of `steps` clears, after the launch's own `tiles` workgroups
static EmbedFill embed_fill_part(void* grad, int64_t pieces, int step, int steps, int tiles) {
    const int64_t lo = pieces * step / steps, hi = pieces * (step + 1) / steps;
    EmbedFill f;
    f.base = (uint4*)grad + lo;
    f.count = hi - lo;
    f.first = tiles;
    const int64_t blocks = (f.count + 2047) / 2048;             // 32 KB each
    f.blocks = (int)(blocks < 8192 ? blocks : 8192);
    return f;
}
template <int BITS, class Src>
static int embed_pass(Src src, int n, unsigned shift, void* hist, uint2* out, void* grad, int64_t pieces,
                      int* step, int steps, hipStream_t st) {
    const int tiles = (n + SRT_TILE - 1) / SRT_TILE;
    uint16_t* h = nullptr;
    if (tiles > SRT_DIRECT_TILES) {
        h = (uint16_t*)hist;
        const EmbedFill f = embed_fill_part(grad, pieces, (*step)++, steps, tiles);
        DR_LAUNCH_NAMED("embed_hist_kernel", (embed_hist_kernel<BITS, Src>), dim3(tiles + f.blocks), dim3(SRT_T), 0, st, src, n,
                        shift, h, f);
        DR_CHECK_LAUNCH("embed_hist_kernel");
    }
    const EmbedFill f = embed_fill_part(grad, pieces, (*step)++, steps, tiles);
    DR_LAUNCH_NAMED("embed_scatter_kernel", (embed_scatter_kernel<BITS, Src>), dim3(tiles + f.blocks), dim3(SRT_T), 0, st, src, n,
                    shift, (const uint16_t*)h, tiles, out, f);
    DR_CHECK_LAUNCH("embed_scatter_kernel");
    return DR_OK;
}
template <class Src>
static int embed_pass_bits(unsigned bits, Src src, int n, unsigned shift, void* hist, uint2* out, void* grad,
                           int64_t pieces, int* step, int steps, hipStream_t st) {
    switch (bits) {
        case 8: return embed_pass<8>(src, n, shift, hist, out, grad, pieces, step, steps, st);
        case 9: return embed_pass<9>(src, n, shift, hist, out, grad, pieces, step, steps, st);
        case 10: return embed_pass<10>(src, n, shift, hist, out, grad, pieces, step, steps, st);
        default: return embed_pass<11>(src, n, shift, hist, out, grad, pieces, step, steps, st);
    }
}

template <class T, class Id>
static int embed_backward_t(int dt, const void* gout, const void* ids, int64_t n, int64_t rows, int d, float scale,
                            int64_t padding, void* grad, char* ws, hipStream_t st) {
    const EmbedLayout L = embed_layout(n, d);
    constexpr int VZ = 16 / (int)sizeof(T);
    const int64_t pieces = rows * d / VZ;                          // and fewer than VZ elements behind them
    const int n_tail = (int)(rows * d - pieces * VZ);
    const bool own_sort = n > 0 && n <= SRT_MAX_N;
    if (!own_sort || n_tail > 0) {
        EmbedFill f = embed_fill_part(grad, own_sort ? 0 : pieces, 0, 1, 0);
        if (f.blocks < 1) f.blocks = 1;
        DR_LAUNCH_NAMED("embed_zero_kernel", (embed_zero_kernel<T>), dim3(f.blocks), dim3(256), 0, st, f, (T*)grad + pieces * VZ,
                        n_tail);
        DR_CHECK_LAUNCH("embed_zero_kernel");
    }
    if (n == 0) return DR_OK;
    EmbedArgs a;
    a.n = n;
    a.rows = rows;
    a.chunk = embed_chunk(n);
    a.chunks = (n + a.chunk - 1) / a.chunk;
    a.d = d;
    a.scale = scale;
    a.part = (float*)(ws + L.part);
    a.state = (uint8_t*)(ws + L.state);
    uint2 *pa = (uint2*)(ws + L.pairs_a), *pb = (uint2*)(ws + L.pairs_b);
    const EmbedKeys<Id> src{(const Id*)ids, rows, padding};
    if (own_sort) {
        unsigned bits, passes;
        embed_digits(rows, &bits, &passes);
        const int steps = (int)passes * ((n + SRT_TILE - 1) / SRT_TILE > SRT_DIRECT_TILES ? 2 : 1);
        int step = 0;
        for (unsigned q = 0; q < passes; ++q) {
            const int rc = q == 0 ? embed_pass_bits(bits, src, (int)n, 0, ws + L.hist, pb, grad, pieces, &step, steps, st)
                                  : embed_pass_bits(bits, EmbedPairs{pa}, (int)n, q * bits, ws + L.hist, pb, grad, pieces,
                                                    &step, steps, st);
            if (rc != DR_OK) return rc;
            std::swap(pa, pb);
        }
        a.keys = (const uint32_t*)pa;
        a.spos = a.keys + 1;
        a.step = 2;
    } else {
        unsigned end_bit = 1;
        while (end_bit < 32 && ((uint64_t)rows >> end_bit) != 0) ++end_bit;     // the sentinel `rows` included
        uint32_t *ka = (uint32_t*)pa, *kb = (uint32_t*)pb;                      // keys, then positions
        const int rc = lsd_sort(src, n, end_bit, ka, (int32_t*)(ka + n), kb, (int32_t*)(kb + n), ws + L.hist,
                                (int32_t*)nullptr, st);
        if (rc != DR_OK) return rc;
        a.keys = kb;
        a.spos = kb + n;
        a.step = 1;
    }
    switch (embed_width(dt, d, gout, grad)) {
        case 8:
            if constexpr (sizeof(T) == 2) return embed_sum_v<T, 8>(a, gout, grad, st);
        case 4: return embed_sum_v<T, 4>(a, gout, grad, st);
        case 2: return embed_sum_v<T, 2>(a, gout, grad, st);
        default: return embed_sum_v<T, 1>(a, gout, grad, st);
    }
}
}  // namespace dr

extern "C" int32_t dr_embed_forward(const void* table, int64_t rows, int32_t d, int32_t dtype, const void* ids, int64_t n,
                                    int32_t id_bits, float scale, void* out, void* stream) {
    using namespace dr;
    DR_REQUIRE(dtype_ok(dtype), "dr_embed_forward: dtype %d", dtype);
    DR_REQUIRE(id_bits == 32 || id_bits == 64, "dr_embed_forward: id_bits must be 32 or 64");
    DR_REQUIRE(n >= 0 && n < (1ll << 40) && rows >= 1 && rows < (1ll << 40) && d >= 1 && d <= EMB_MAX_D,
               "dr_embed_forward: bad sizes (n=%lld rows=%lld d=%d)", (long long)n, (long long)rows, d);
    if (n == 0) return DR_OK;
    DR_REQUIRE(table && ids && out, "dr_embed_forward: NULL pointer");
    DR_REQUIRE(aligned_to(table, dtype_size(dtype)) && aligned_to(out, dtype_size(dtype)) && aligned_to(ids, id_bits / 8),
               "dr_embed_forward: a pointer is not aligned to its element size");
    hipStream_t st = (hipStream_t)stream;
#define EMB_FWD(T)                                                                                                    \
    return id_bits == 32 ? embed_forward_t<T, int32_t>(dtype, table, rows, d, ids, n, scale, out, st)                 \
                         : embed_forward_t<T, int64_t>(dtype, table, rows, d, ids, n, scale, out, st)
    DR_BY_DTYPE(dtype, EMB_FWD);
#undef EMB_FWD
}

extern "C" int64_t dr_embed_backward_bytes(int64_t n, int32_t d) {
    if (n < 0 || n >= (1ll << 31) - dr::LSD_TILE || d < 1 || d > dr::EMB_MAX_D) return DR_ERR_ARG;
    return dr::embed_layout(n, d).total + 256;
}

extern "C" int32_t dr_embed_backward(const void* gout, int64_t n, int32_t d, int32_t dtype, const void* ids, int32_t id_bits,
                                     int64_t rows, float scale, int64_t padding, void* grad, void* ws, int64_t ws_bytes,
                                     void* stream) {
    using namespace dr;
    DR_REQUIRE(dtype_ok(dtype), "dr_embed_backward: dtype %d", dtype);
    DR_REQUIRE(id_bits == 32 || id_bits == 64, "dr_embed_backward: id_bits must be 32 or 64");
    DR_REQUIRE(n >= 0 && n < (1ll << 31) - LSD_TILE && rows >= 1 && rows < (1ll << 31) - 1 && d >= 1 && d <= EMB_MAX_D,
               "dr_embed_backward: bad sizes (n=%lld rows=%lld d=%d)", (long long)n, (long long)rows, d);
    DR_REQUIRE(grad && (n == 0 || (gout && ids)), "dr_embed_backward: NULL pointer");
    DR_REQUIRE(aligned_to(grad, 16), "dr_embed_backward: grad must be 16-byte aligned");
    DR_REQUIRE(aligned_to(gout, dtype_size(dtype)) && aligned_to(ids, id_bits / 8),
               "dr_embed_backward: a pointer is not aligned to its element size");
    DR_REQUIRE(n == 0 || (ws && aligned_to(ws, 256)), "dr_embed_backward: workspace is NULL or not 256-byte aligned");
    if (n > 0 && ws_bytes < dr_embed_backward_bytes(n, d))
        DR_FAIL(DR_ERR_WORKSPACE, "dr_embed_backward: workspace %lld < required %lld", (long long)ws_bytes,
                (long long)dr_embed_backward_bytes(n, d));
    hipStream_t st = (hipStream_t)stream;
#define EMB_BWD(T)                                                                                                     \
    return id_bits == 32                                                                                               \
               ? embed_backward_t<T, int32_t>(dtype, gout, ids, n, rows, d, scale, padding, grad, (char*)ws, st)       \
               : embed_backward_t<T, int64_t>(dtype, gout, ids, n, rows, d, scale, padding, grad, (char*)ws, st)
    DR_BY_DTYPE(dtype, EMB_BWD);
#undef EMB_BWD
}
