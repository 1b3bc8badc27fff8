// Embedding lookup with scaling, fp32 / fp16 / bf16 tables, and its gradient by sorted ids.
//   forward   out[e, :] = scale * table[ids[e], :]            (an id outside [0, rows): a zero row, as dr_gather_f32)
//   backward  grad[r, :] = scale * sum over e with ids[e] == r of gout[e, :]   for EVERY row r (untouched rows: 0);
//             ids equal to padding, or outside [0, rows), contribute nothing.
// HBM-bound both ways.  Sums are fp32 in a fixed order (sorted list cut into blocks of EMB_CHUNK entries, entries in list
// order inside a block, a row's blocks in ascending order): the same ids and gradients give the same bits, with no atomics.
#include "dr_lsd_sort.h"
#include "dr_types.h"

namespace dr {

constexpr int EMB_MAX_D = 32768;
constexpr int EMB_CHUNK = 32;        // sorted entries a group of lanes sums
constexpr int EMB_DEPTH = 8;         // gradient rows of a chunk in flight per lane group
constexpr int64_t EMB_SMALL_N = 4096;   // lists the one-workgroup plan sorts in one launch (segment.hip)

// ---- forward -------------------------------------------------------------------------------------------------------
// A block owns R whole rows = R * cpr vectors of V elements, dealt to its threads in order, so every lane moves 16 bytes
// (or the widest piece the row size and the bases allow) whatever d is; U independent id -> row chains per thread.
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

template <class T>
__global__ __launch_bounds__(256) void embed_zero_kernel(T* __restrict__ grad, int64_t count) {
    constexpr int V = 16 / (int)sizeof(T);
    typename VecType<T, V>::type z;
#pragma unroll
    for (int x = 0; x < V; ++x) z[x] = (T)0.0f;
    const int64_t nv = count / V, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nv; i += step)
        *reinterpret_cast<typename VecType<T, V>::type*>(grad + i * V) = z;
    if (blockIdx.x == 0 && threadIdx.x < (unsigned)(count - nv * V)) grad[nv * V + threadIdx.x] = (T)0.0f;
}

struct EmbedArgs {
    const uint32_t* keys;   // sorted keys (>= rows: contributes nothing), or NULL: looked up through ids
    const int32_t* spos;    // sorted list positions
    const void* ids;
    int64_t n, rows, padding, chunks;
    int d;
    float scale;
    float* part;            // [chunks, 2, d] sums of the runs that cross a chunk border: first run, last run
};

template <class Id>
__device__ __forceinline__ int64_t embed_key(const EmbedArgs& a, int64_t s) {
    if (a.keys) return (int64_t)a.keys[s];
    const int64_t id = (int64_t)((const Id*)a.ids)[a.spos[s]];
    return (id < 0 || id >= a.rows || id == a.padding) ? a.rows : id;
}

// One group of LPR lanes per chunk.  A run (equal keys) that lies inside the chunk is finished here; the part of a run that
// began in an earlier chunk goes to part[chunk][0], the part of one that goes on behind the chunk to part[chunk][1] (a run
// that does both: [0]).
template <class T, class Id, int V, int LPR>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedArgs a, const T* __restrict__ gout, T* __restrict__ grad) {
    const int64_t chunk = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
    if (chunk >= a.chunks) return;
    const int lane = threadIdx.x % LPR;
    const int64_t s0 = chunk * EMB_CHUNK;
    const int m = (int)(a.n - s0 < EMB_CHUNK ? a.n - s0 : EMB_CHUNK);
    if (a.keys && a.keys[s0] >= (uint32_t)a.rows) return;    // sorted: nothing from here on contributes
    const int64_t before = s0 > 0 ? embed_key<Id>(a, s0 - 1) : -1, behind = s0 + m < a.n ? embed_key<Id>(a, s0 + m) : -1;
    for (int c = lane * V; c < a.d; c += LPR * V) {
        float acc[V];
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] = 0.0f;
        int64_t run = -1;                          // key of the run being summed
        bool carried = false;                      // it began before this chunk
        for (int q0 = 0; q0 < m; q0 += EMB_DEPTH) {
            int64_t key[EMB_DEPTH];
            float v[EMB_DEPTH][V];
#pragma unroll
            for (int q = 0; q < EMB_DEPTH; ++q) {
                const int64_t s = s0 + (q0 + q < m ? q0 + q : m - 1);
                key[q] = embed_key<Id>(a, s);
                load_f32<T, V>(v[q], gout + (int64_t)a.spos[s] * a.d + c);
            }
#pragma unroll
            for (int q = 0; q < EMB_DEPTH; ++q) {
                if (q0 + q >= m || key[q] >= a.rows) continue;
                if (key[q] != run) {
                    if (run >= 0) {
                        if (carried) {
                            store_f32<float, V>(a.part + (chunk * 2) * a.d + c, acc);
                        } else {
#pragma unroll
                            for (int x = 0; x < V; ++x) acc[x] *= a.scale;
                            store_f32<T, V>(grad + run * a.d + c, acc);
                        }
                    }
                    run = key[q];
                    carried = q0 + q == 0 && before == run;
#pragma unroll
                    for (int x = 0; x < V; ++x) acc[x] = 0.0f;
                }
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] += v[q][x];
            }
        }
        if (run < 0) continue;
        if (carried) {
            store_f32<float, V>(a.part + (chunk * 2) * a.d + c, acc);
        } else if (behind == run) {
            store_f32<float, V>(a.part + (chunk * 2 + 1) * a.d + c, acc);
        } else {
#pragma unroll
            for (int x = 0; x < V; ++x) acc[x] *= a.scale;
            store_f32<T, V>(grad + run * a.d + c, acc);
        }
    }
}

// Joins the runs that cross chunk borders: one block per chunk in which such a run BEGINS; the 256 threads of the block
// are 256 / LPR groups that take every (256 / LPR)-th of the run's chunks, the groups' sums are added in order.
template <class T, class Id, int V, int LPR>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedArgs a, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / LPR;
    __shared__ float red[GROUPS][LPR * V];
    __shared__ int64_t run_s;
    __shared__ int64_t last_s;
    for (int64_t chunk = blockIdx.x; chunk + 1 < a.chunks; chunk += gridDim.x) {
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t s0 = chunk * EMB_CHUNK, e = s0 + EMB_CHUNK;          // e < n: not the last chunk
            const int64_t run = embed_key<Id>(a, e - 1);
            bool begins = run < a.rows && embed_key<Id>(a, e) == run;
            if (begins && embed_key<Id>(a, s0) == run && s0 > 0 && embed_key<Id>(a, s0 - 1) == run) begins = false;
            run_s = begins ? run : -1;
            if (begins) {                                                       // last chunk the run reaches
                int64_t lo = chunk + 1, hi = a.chunks - 1;
                while (lo < hi) {
                    const int64_t mid = (lo + hi + 1) >> 1;
                    if (embed_key<Id>(a, mid * EMB_CHUNK) == run) lo = mid; else hi = mid - 1;
                }
                last_s = lo;
            }
        }
        __syncthreads();
        const int64_t run = run_s;
        if (run < 0) continue;                                                  // block-uniform
        const int64_t last = last_s;
        const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
        for (int c0 = 0; c0 < a.d; c0 += LPR * V) {
            const int c = c0 + lane * V;
            float acc[V];
#pragma unroll
            for (int x = 0; x < V; ++x) acc[x] = 0.0f;
            if (c < a.d)
#pragma unroll 4
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
#pragma unroll
                for (int g = 1; g < GROUPS; ++g)
#pragma unroll
                    for (int x = 0; x < V; ++x) acc[x] += red[g][lane * V + x];
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] *= a.scale;
                store_f32<T, V>(grad + run * a.d + c, acc);
            }
            __syncthreads();
        }
    }
}

struct EmbedLayout {
    int64_t keys_a, keys_b, vals_a, vals_b, hdr, lsd, plan, part, total;
};
static EmbedLayout embed_layout(int64_t n, int d) {
    EmbedLayout L;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = off;
        off += align_up(bytes, 256);
        return o;
    };
    L.keys_a = L.keys_b = L.vals_a = L.vals_b = L.hdr = L.lsd = L.plan = 0;
    if (n <= EMB_SMALL_N) {
        L.plan = take(dr_segment_plan_bytes(n, 1));
    } else {
        L.keys_a = take(n * 4);
        L.keys_b = take(n * 4);
        L.vals_a = take(n * 4);
        L.vals_b = take(n * 4);
        L.lsd = take(lsd_scratch_bytes(n));
    }
    L.part = take((n + EMB_CHUNK - 1) / EMB_CHUNK * 2 * (int64_t)d * 4);
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
    // rows per block: up to 2048 pieces (8 per thread), fewer while that leaves less than 4 blocks per CU
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

template <class T, class Id, int V, int LPR>
static int embed_sum_launch(const EmbedArgs& a, const void* gout, void* grad, hipStream_t st) {
    const int64_t blocks = (a.chunks * LPR + 255) / 256;
    DR_REQUIRE(blocks < (1ll << 31), "dr_embed_backward: too many blocks");
    DR_LAUNCH_NAMED("embed_sum_kernel", (embed_sum_kernel<T, Id, V, LPR>), dim3((unsigned)blocks), dim3(256), 0, st, a,
                    (const T*)gout, (T*)grad);
    DR_CHECK_LAUNCH("embed_sum_kernel");
    if (a.chunks > 1) {
        const int grid = (int)(a.chunks - 1 < 4096 ? a.chunks - 1 : 4096);
        DR_LAUNCH_NAMED("embed_join_kernel", (embed_join_kernel<T, Id, V, LPR>), dim3(grid), dim3(256), 0, st, a, (T*)grad);
        DR_CHECK_LAUNCH("embed_join_kernel");
    }
    return DR_OK;
}
template <class T, class Id, int V>
static int embed_sum_v(const EmbedArgs& a, const void* gout, void* grad, hipStream_t st) {
    const int cpr = a.d / V;
    if (cpr <= 4) return embed_sum_launch<T, Id, V, 4>(a, gout, grad, st);
    if (cpr <= 8) return embed_sum_launch<T, Id, V, 8>(a, gout, grad, st);
    if (cpr <= 16) return embed_sum_launch<T, Id, V, 16>(a, gout, grad, st);
    if (cpr <= 32) return embed_sum_launch<T, Id, V, 32>(a, gout, grad, st);
    return embed_sum_launch<T, Id, V, 64>(a, gout, grad, st);
}

template <class T, class Id>
static int embed_backward_t(int dt, const void* gout, const void* ids, int64_t n, int64_t rows, int d, float scale,
                            int64_t padding, void* grad, char* ws, hipStream_t st) {
    const EmbedLayout L = embed_layout(n, d);
    {
        constexpr int V = 16 / (int)sizeof(T);
        DR_LAUNCH_NAMED("embed_zero_kernel", (embed_zero_kernel<T>), dim3(grid_for(rows * d / V + 1, 256)), dim3(256), 0, st,
                        (T*)grad, rows * d);
        DR_CHECK_LAUNCH("embed_zero_kernel");
    }
    if (n == 0) return DR_OK;
    EmbedArgs a;
    a.ids = ids;
    a.n = n;
    a.rows = rows;
    a.padding = padding;
    a.chunks = (n + EMB_CHUNK - 1) / EMB_CHUNK;
    a.d = d;
    a.scale = scale;
    a.part = (float*)(ws + L.part);
    if (n <= EMB_SMALL_N) {
        int rc = dr_segment_plan(ids, n, (int)sizeof(Id) * 8, rows, ws + L.plan, dr_segment_plan_bytes(n, 1), st);
        if (rc != DR_OK) return rc;
        rc = dr_segment_plan_view(ws + L.plan, n, &a.spos, nullptr, nullptr, nullptr);
        if (rc != DR_OK) return rc;
        a.keys = nullptr;
    } else {
        unsigned end_bit = 1;
        while (end_bit < 32 && ((uint64_t)rows >> end_bit) != 0) ++end_bit;     // the sentinel `rows` included
        const int rc = lsd_sort(EmbedKeys<Id>{(const Id*)ids, rows, padding}, n, end_bit, (uint32_t*)(ws + L.keys_a),
                                (int32_t*)(ws + L.vals_a), (uint32_t*)(ws + L.keys_b), (int32_t*)(ws + L.vals_b), ws + L.lsd,
                                (int32_t*)nullptr, st);
        if (rc != DR_OK) return rc;
        a.keys = (const uint32_t*)(ws + L.keys_b);
        a.spos = (const int32_t*)(ws + L.vals_b);
    }
    switch (embed_width(dt, d, gout, grad)) {
        case 8:
            if constexpr (sizeof(T) == 2) return embed_sum_v<T, Id, 8>(a, gout, grad, st);
        case 4: return embed_sum_v<T, Id, 4>(a, gout, grad, st);
        case 2: return embed_sum_v<T, Id, 2>(a, gout, grad, st);
        default: return embed_sum_v<T, Id, 1>(a, gout, grad, st);
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
