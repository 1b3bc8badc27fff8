// Global norm of a list of gradients and the list scaled to it (tf.clip_by_global_norm):
//   n = sqrt(sum over all tensors and elements of t^2),  out = t * clip_norm / max(n, clip_norm)
// (a non-finite n makes every output NaN, as there).  HBM-bound: the norm has to be known before the first output, so
// the least traffic is two reads and one write of everything.
//
// Two launches per 128 tensors, whatever their number and sizes: the tensors are cut into chunks of 8192 elements that
// all blocks walk together, so a hundred odd-sized weights cost no more launches than one table.  The tensor list
// travels in the kernel arguments (no device table to upload: the call can be captured into a graph).
//   clip_norm_kernel   a block's sum of squares in fp64 -- no overflow or underflow for any fp32 value, and the sum of
//                      10^9 squares keeps 40 bits -- to one slot per block: a fixed order, no atomics.
//   clip_scale_kernel  every block adds up the slots itself (at most 1024 per 128 tensors, from L2: cheaper than a third
//                      launch), then scales its chunks, LAST chunk first: what the norm pass read last is still in the
//                      256 MB Infinity Cache.
// 54 tensors of 141 MB in mixed types: norm 24 us = 5.9 TB/s, scaling 45 us = 6.3 TB/s; 12 small tensors: 4.2 + 4.6 us.
#include <algorithm>
#include <new>

#include "dr_types.h"

namespace dr {

constexpr int CLIP_TENSORS = 128;    // per launch: 128 x 24 bytes + chunk table fit the 4 KB of kernel arguments
constexpr int CLIP_CHUNK = 8192;     // elements: 32 KB (16 KB) per block and step, 8 (4) 16-byte loads per thread
constexpr int CLIP_BLOCKS = 1024;    // 4 blocks of 256 threads per CU, 8 loads of 16 bytes in flight each

struct ClipArgs {
    const void* in[CLIP_TENSORS];
    void* out[CLIP_TENSORS];
    int64_t count[CLIP_TENSORS];
    int32_t first[CLIP_TENSORS + 1];   // first chunk of tensor i; [n] = number of chunks
    uint8_t dtype[CLIP_TENSORS];       // DR_F32 / DR_F16 / DR_BF16
    int32_t n;
};
static_assert(sizeof(ClipArgs) <= 3800, "ClipArgs travels in the kernel arguments");

__device__ __forceinline__ int clip_tensor_of(const ClipArgs& a, int chunk) {
    int lo = 0, hi = a.n - 1;                       // last tensor whose first chunk is <= chunk (empty ones own none)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// sum of squares of one chunk by 256 threads: 16-byte loads issued together, two fp64 accumulators a thread
template <class T>
__device__ __forceinline__ void chunk_squares(const T* p, int len, double& s0, double& s1) {
    constexpr int V = 16 / (int)sizeof(T), ROUNDS = CLIP_CHUNK / (256 * V);
    if (len == CLIP_CHUNK && ((uintptr_t)p & 15) == 0) {
        float r[ROUNDS][V];
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) load_f32<T, V>(r[q], p + ((int)threadIdx.x + q * 256) * V);
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q)
#pragma unroll
            for (int x = 0; x < V; x += 2) {
                s0 = fma((double)r[q][x], (double)r[q][x], s0);
                s1 = fma((double)r[q][x + 1], (double)r[q][x + 1], s1);
            }
        return;
    }
    int e = 0;
    if (((uintptr_t)p & 15) == 0) {                 // a ragged last chunk: vectors, then single elements
        e = len / V * V;
        for (int i = (int)threadIdx.x * V; i < e; i += 256 * V) {
            float r[V];
            load_f32<T, V>(r, p + i);
#pragma unroll
            for (int x = 0; x < V; x += 2) {
                s0 = fma((double)r[x], (double)r[x], s0);
                s1 = fma((double)r[x + 1], (double)r[x + 1], s1);
            }
        }
    }
#pragma unroll 8
    for (int i = e + (int)threadIdx.x; i < len; i += 256) {
        const double v = (double)(float)p[i];
        s0 = fma(v, v, s0);
    }
}

template <class T>
__device__ __forceinline__ void chunk_scale(const T* p, T* o, int len, float c) {
    constexpr int V = 16 / (int)sizeof(T), ROUNDS = CLIP_CHUNK / (256 * V);
    const bool vec = (((uintptr_t)p | (uintptr_t)o) & 15) == 0;
    if (len == CLIP_CHUNK && vec) {
        float r[ROUNDS][V];
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) load_f32<T, V>(r[q], p + ((int)threadIdx.x + q * 256) * V);
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) {
#pragma unroll
            for (int x = 0; x < V; ++x) r[q][x] *= c;
            store_f32<T, V>(o + ((int)threadIdx.x + q * 256) * V, r[q]);
        }
        return;
    }
    int e = 0;
    if (vec) {
        e = len / V * V;
        for (int i = (int)threadIdx.x * V; i < e; i += 256 * V) {
            float r[V];
            load_f32<T, V>(r, p + i);
#pragma unroll
            for (int x = 0; x < V; ++x) r[x] *= c;
            store_f32<T, V>(o + i, r);
        }
    }
#pragma unroll 8
    for (int i = e + (int)threadIdx.x; i < len; i += 256) o[i] = (T)((float)p[i] * c);
}

// sum of one double per thread over the 256 threads of a block, in a fixed order; every thread gets it
__device__ __forceinline__ double block_sum_f64(double s, double* red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return ((red[0] + red[1]) + red[2]) + red[3];
}

__global__ __launch_bounds__(256) void clip_norm_kernel(ClipArgs a, double* __restrict__ slots) {
    __shared__ double red[4];
    double s0 = 0.0, s1 = 0.0;
    const int chunks = a.first[a.n];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = clip_tensor_of(a, c);
        const int64_t off = (int64_t)(c - a.first[t]) * CLIP_CHUNK, left = a.count[t] - off;
        const int len = left < CLIP_CHUNK ? (int)left : CLIP_CHUNK;
        if (a.dtype[t] == DR_F32)
            chunk_squares((const float*)a.in[t] + off, len, s0, s1);
        else if (a.dtype[t] == DR_F16)
            chunk_squares((const f16*)a.in[t] + off, len, s0, s1);
        else
            chunk_squares((const bf16*)a.in[t] + off, len, s0, s1);
    }
    const double s = block_sum_f64(s0 + s1, red);
    if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

// nslots slots -> the norm; norm_out (NULL: not here) gets it from block 0.  scale = 0: only the norm is wanted.
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipArgs a, const double* __restrict__ slots, int nslots,
                                                         float clip_norm, float* __restrict__ norm_out, int scale) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < nslots; i += 256) s += slots[i];
    const double norm = sqrt(block_sum_f64(s, red));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    if (!scale) return;
    const double lim = (double)clip_norm;
    // inf - inf and NaN - NaN are NaN, anything finite gives 0
    const float c = (norm - norm == 0.0) ? (float)(lim / (norm > lim ? norm : lim)) : __builtin_nanf("");
    const int chunks = a.first[a.n];
    for (int q = blockIdx.x; q < chunks; q += gridDim.x) {
        const int ch = chunks - 1 - q;
        const int t = clip_tensor_of(a, ch);
        if (c == 1.0f && a.out[t] == a.in[t]) continue;              // in place and nothing to clip
        const int64_t off = (int64_t)(ch - a.first[t]) * CLIP_CHUNK, left = a.count[t] - off;
        const int len = left < CLIP_CHUNK ? (int)left : CLIP_CHUNK;
        if (a.dtype[t] == DR_F32)
            chunk_scale((const float*)a.in[t] + off, (float*)a.out[t] + off, len, c);
        else if (a.dtype[t] == DR_F16)
            chunk_scale((const f16*)a.in[t] + off, (f16*)a.out[t] + off, len, c);
        else
            chunk_scale((const bf16*)a.in[t] + off, (bf16*)a.out[t] + off, len, c);
    }
}

namespace {
struct Range {
    uintptr_t lo, hi;
    int32_t i;
    bool out;
    bool operator<(const Range& o) const { return lo < o.lo; }
};
// An output may be its own input; any other overlap of an output would be a race.  Returns the offending index or -1.
int clip_overlap(const void* const* in, void* const* out, const int64_t* count, const int32_t* dt, int32_t n, Range* r) {
    int m = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (count[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)(count[i] * dtype_size(dt[i]));
        r[m++] = Range{(uintptr_t)out[i], (uintptr_t)out[i] + bytes, i, true};
        if (in[i] != out[i]) r[m++] = Range{(uintptr_t)in[i], (uintptr_t)in[i] + bytes, i, false};
    }
    std::sort(r, r + m);
    uintptr_t end_out = 0, end_in = 0;               // furthest end of the outputs / inputs seen so far
    for (int q = 0; q < m; ++q) {
        if (r[q].lo < end_out || (r[q].out && r[q].lo < end_in)) return r[q].i;
        uintptr_t& e = r[q].out ? end_out : end_in;
        if (r[q].hi > e) e = r[q].hi;
    }
    return -1;
}
}  // namespace
}  // namespace dr

extern "C" int64_t dr_global_norm_bytes(int32_t n) {
    if (n < 0) return DR_ERR_ARG;
    const int64_t launches = (n + dr::CLIP_TENSORS - 1) / dr::CLIP_TENSORS;
    return dr::align_up((launches > 0 ? launches : 1) * dr::CLIP_BLOCKS * (int64_t)sizeof(double), 256);
}

extern "C" int32_t dr_clip_global_norm(const void* const* in, void* const* out, const int64_t* count,
                                       const int32_t* dtype, int32_t n, float clip_norm, float* norm_out, void* ws,
                                       int64_t ws_bytes, void* stream) {
    using namespace dr;
    DR_REQUIRE(n >= 0 && (n == 0 || (in && count && dtype)), "dr_clip_global_norm: bad tensor list");
    DR_REQUIRE(out != nullptr || norm_out != nullptr, "dr_clip_global_norm: neither out nor norm_out is wanted");
    DR_REQUIRE(out == nullptr || (clip_norm > 0.0f && clip_norm <= 3.402823466e38f),
               "dr_clip_global_norm: clip_norm must be positive and finite");
    DR_REQUIRE(ws != nullptr && aligned_to(ws, 8), "dr_clip_global_norm: workspace is NULL or misaligned");
    if (ws_bytes < dr_global_norm_bytes(n))
        DR_FAIL(DR_ERR_WORKSPACE, "dr_clip_global_norm: workspace %lld < required %lld", (long long)ws_bytes,
                (long long)dr_global_norm_bytes(n));
    for (int32_t i = 0; i < n; ++i) {
        DR_REQUIRE(dtype_ok(dtype[i]), "dr_clip_global_norm: tensor %d has dtype %d", i, dtype[i]);
        DR_REQUIRE(count[i] >= 0 && count[i] < (1ll << 43), "dr_clip_global_norm: tensor %d has %lld elements", i,
                   (long long)count[i]);
        DR_REQUIRE(count[i] == 0 || (in[i] && (!out || out[i])), "dr_clip_global_norm: tensor %d is NULL", i);
        DR_REQUIRE(count[i] == 0 || (aligned_to(in[i], dtype_size(dtype[i])) && (!out || aligned_to(out[i], dtype_size(dtype[i])))),
                   "dr_clip_global_norm: tensor %d is not aligned to its element size", i);
    }
    if (out != nullptr && n > 0) {
        Range few[256];
        Range* r = n <= 128 ? few : new (std::nothrow) Range[2 * (size_t)n];
        DR_REQUIRE(r != nullptr, "dr_clip_global_norm: out of host memory");
        const int bad = clip_overlap(in, out, count, dtype, n, r);
        if (r != few) delete[] r;
        DR_REQUIRE(bad < 0, "dr_clip_global_norm: output memory overlaps another tensor's (tensor %d)", bad);
    }
    hipStream_t st = (hipStream_t)stream;
    double* slots = (double*)ws;
    int nslots = 0;
    const int32_t parts = n > 0 ? (n + CLIP_TENSORS - 1) / CLIP_TENSORS : 1;
    for (int pass = 0; pass < 2; ++pass)
        for (int32_t part = 0; part < parts; ++part) {
            ClipArgs a;
            memset(&a, 0, sizeof(a));
            const int32_t t0 = part * CLIP_TENSORS;
            a.n = n - t0 < CLIP_TENSORS ? n - t0 : CLIP_TENSORS;
            int64_t chunks = 0;
            for (int32_t i = 0; i < a.n; ++i) {
                a.in[i] = in[t0 + i];
                a.out[i] = out ? out[t0 + i] : nullptr;
                a.count[i] = count[t0 + i];
                a.dtype[i] = (uint8_t)dtype[t0 + i];
                a.first[i] = (int32_t)chunks;
                chunks += (count[t0 + i] + CLIP_CHUNK - 1) / CLIP_CHUNK;
                DR_REQUIRE(chunks < (1ll << 31) - CLIP_BLOCKS, "dr_clip_global_norm: too many elements");
            }
            for (int32_t i = a.n; i <= CLIP_TENSORS; ++i) a.first[i] = (int32_t)chunks;
            const int grid = chunks < CLIP_BLOCKS ? (int)chunks : CLIP_BLOCKS;
            if (pass == 0) {
                if (grid == 0) continue;
                DR_LAUNCH_NAMED("clip_norm_kernel", clip_norm_kernel, dim3(grid), dim3(256), 0, st, a, slots + nslots);
                DR_CHECK_LAUNCH("clip_norm_kernel");
                nslots += grid;
            } else {
                const bool first = part == 0;
                if (out == nullptr && !first) continue;
                const int g2 = out != nullptr ? (grid > 0 ? grid : (first ? 1 : 0)) : 1;
                if (g2 == 0) continue;
                DR_LAUNCH_NAMED("clip_scale_kernel", clip_scale_kernel, dim3(g2), dim3(256), 0, st, a,
                                (const double*)slots, nslots, clip_norm, first ? norm_out : (float*)nullptr,
                                out != nullptr ? 1 : 0);
                DR_CHECK_LAUNCH("clip_scale_kernel");
            }
        }
    return DR_OK;
}
