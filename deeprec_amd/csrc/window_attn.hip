// Causal attention over a sliding window and the first few items of a history:
//   key j is visible to query i iff begin <= j <= i < end and (i - j < window or j - begin < sinks)
//   out_i = sum_j p_ij v_j,  p_i = softmax_j(scale <q_i, k_j>) over the visible j;   lse_i = log sum_j exp(scale <q_i, k_j>)
// [begin, end) is the part of the row that holds the history (padding on either side); a query outside it gets zeros and
// lse = -inf, and what stands outside reaches no result.  Hq query heads share Hkv key / value heads in groups.
//
// Tiles of 16 queries x 16 keys on the matrix cores.  The contraction is laid out so that nothing moves between lanes: with
// S^T = K Q^T a lane holds, for ONE query, four keys of each 16-key tile (rows 4 g + i of lane group g), and that is already
// the B operand of O^T = V^T P^T if slot (g, e) of the 32-long contraction means key 4 g + e (e < 4) or 16 + 4 g + e - 4:
// the order of a sum is free as long as A uses the same one, and A = V^T is read from LDS by that rule (two transposing
// 8-byte reads for 16-bit types, eight 4-byte reads for fp32).  Running maximum and sum are one scalar per lane.
// fp32 runs the same code: a 16x16x32 step is eight v_mfma_f32_16x16x4_f32, element e of every lane's eight in step e.
// Scores, statistics and sums are fp32.  The second product's operands are of the storage type; P and dS, of 16-bit types, go
// in as two halves (hi + what hi misses): rounded once, P alone put as much error into out and dV as their own rounding, and
// where terms cancel far more.  The second half costs 9 % of the forward at D = 128 (28.5 -> 30.6 us at 4 x 2047 x 8 / 2 heads,
// window 256), 20 % at D = 64 on a large grid, 3 % of dK / dV, nothing for one token.
#include <initializer_list>
#include <type_traits>

#include "dr_types.h"

namespace dr {

constexpr int WA_MAX_D = 256, WA_MAX_SINKS = 64;
constexpr int WA_MAX_SPLITS = 256;
constexpr int64_t WA_MAX_GRID = 1 << 24;   // workgroups of 256: a launch counts its threads in 32 bits
constexpr int WA_BK = 32;              // keys (queries in the dK / dV kernels) per tile
constexpr float WA_LOG2E = 1.44269504088896340736f, WA_LN2 = 0.69314718055994530942f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
template <class T>
using Oct = typename VecType<T, 8>::type;

__device__ __forceinline__ f32x4 mma(const Oct<bf16>& a, const Oct<bf16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Oct<f16>& a, const Oct<f16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Oct<float>& a, const Oct<float>& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// Probabilities go into their products times 2^p_bits, undone in fp32: without, fp16 loses what lies below 2^-14 and drops what
// lies below 2^-25, and with it the whole gradient of keys that no query weighs strongly.  (The 15 is added to the exponent:
// its last bit there costs p 2^-21 ln 2, five units of fp32's rounding.)
template <class T>
constexpr float p_bits() {
    return std::is_same<T, f16>::value ? 15.0f : 0.0f;
}
template <class T>
constexpr float p_down() {
    return std::is_same<T, f16>::value ? 0x1p-15f : 1.0f;
}
// 2^x of a weight that goes into a product
template <class T>
__device__ __forceinline__ float weight(float d, float c) {
    return __builtin_amdgcn_exp2f(p_bits<T>() == 0.0f ? d * c : fmaf(d, c, p_bits<T>()));
}

// LDS row length: rows of a 16-lane read start 4 banks apart
template <class T, int DP>
constexpr int lds_ld() {
    return DP + (sizeof(T) == 2 ? 8 : 4);
}

// How rows are read: in pieces of 16 bytes (D a multiple of 8, every row start on the 16-byte grid), in words of 4, or one
// 16-bit element at a time.  Loads are never under a condition -- each would wait for the one before -- but go to a clamped
// place, and what does not exist is cleared when the value is used.
enum { WA_PIECES = 0, WA_WORDS = 1, WA_ELEMS = 2 };
template <class T>
__device__ __forceinline__ Oct<T> load_oct(const T* row, int c, int D, int mode) {
    Oct<T> r;
    if (mode == WA_PIECES) {
        const T* p = row + (c < D ? c : 0);
        if constexpr (sizeof(T) == 2) {
            r = *reinterpret_cast<const Oct<T>*>(p);
        } else {
            const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[e] = x[e];
                r[4 + e] = y[e];
            }
        }
    } else if (sizeof(T) == 4 || mode == WA_WORDS) {            // D is even for 16-bit types
        constexpr int N = (int)sizeof(T) * 2, P = 4 / (int)sizeof(T);   // words, elements per word
        typedef uint32_t words __attribute__((ext_vector_type(N)));
        words w;
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = *reinterpret_cast<const uint32_t*>(row + (c + e * P < D ? c + e * P : 0));
        r = __builtin_bit_cast(Oct<T>, w);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = row[c + e < D ? c + e : 0];
    }
    return r;
}
// the first n elements, zeros behind them (pieces: all or nothing)
template <class T>
__device__ __forceinline__ Oct<T> keep_oct(const Oct<T>& r, int n, int mode) {
    constexpr int N = (int)sizeof(T) * 2;
    typedef uint32_t words __attribute__((ext_vector_type(N)));
    if (mode == WA_PIECES) {
        words w = __builtin_bit_cast(words, r);
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = n > 0 ? w[e] : 0u;
        return __builtin_bit_cast(Oct<T>, w);
    }
    Oct<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = e < n ? r[e] : (T)0.0f;
    return o;
}
__device__ __forceinline__ int clamp_row(int row, int lo, int hi) {   // a row that exists, inside [lo, hi) if that is not empty
    if (hi <= lo) return 0;
    return row < lo ? lo : (row >= hi ? hi - 1 : row);
}
template <class T>
__device__ __forceinline__ void lds_store_oct(T* p, const Oct<T>& r) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<Oct<T>*>(p) = r;
    } else {
        *reinterpret_cast<f32x4*>(p) = f32x4{r[0], r[1], r[2], r[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{r[4], r[5], r[6], r[7]};
    }
}
// 8 consecutive elements of a row (operand whose contraction runs along the row)
template <class T>
__device__ __forceinline__ Oct<T> row_frag(const T* p) {
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const Oct<T>*>(p);
    } else {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
        Oct<T> r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[e] = x[e];
            r[4 + e] = y[e];
        }
        return r;
    }
}
// column col0 + (lane & 15) at the 8 rows of lane group g = lane / 16: 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3
template <class T, int LD>
__device__ __forceinline__ Oct<T> col_frag(const T* tile, int col0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    if constexpr (sizeof(T) == 2) {
        // the transposing read: of the 16 lanes of a group, lanes 4 r .. 4 r + 3 name row r's 16 columns, lane i gets
        // column i of the four rows
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const T* p = tile + (4 * g + (i >> 2)) * LD + col0 + 4 * (i & 3);
        struct {
            s16x4 a, b;
        } r;
        r.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
        r.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * LD));
        return __builtin_bit_cast(Oct<T>, r);
    } else {
        Oct<T> r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[e] = tile[(4 * g + e) * LD + col0 + i];
            r[4 + e] = tile[(16 + 4 * g + e) * LD + col0 + i];
        }
        return r;
    }
}
template <class T>
__device__ __forceinline__ Oct<T> to_oct(const f32x4& a, const f32x4& b) {
    Oct<T> r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r[e] = (T)a[e];
        r[4 + e] = (T)b[e];
    }
    return r;
}

// 16-bit operands in two halves: the rounded value and what it misses, e^2 left of it (e: half a step)
template <class T>
__device__ __forceinline__ void split_oct(const f32x4& a, const f32x4& b, Oct<T>& hi, Oct<T>& lo) {
    hi = to_oct<T>(a, b);
    f32x4 x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = a[e] - (float)hi[e];
        y[e] = b[e] - (float)hi[4 + e];
    }
    lo = to_oct<T>(x, y);
}
// over the four lane groups that share a query: every lane gets the maximum / the sum
__device__ __forceinline__ float groups_max(float x) {
    const int lane = threadIdx.x & 63;
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_ds_bpermute((lane ^ 16) << 2, __float_as_int(x))));
    return fmaxf(x, __int_as_float(__builtin_amdgcn_ds_bpermute((lane ^ 32) << 2, __float_as_int(x))));
}
__device__ __forceinline__ float groups_sum(float x) {
    const int lane = threadIdx.x & 63;
    x += __int_as_float(__builtin_amdgcn_ds_bpermute((lane ^ 16) << 2, __float_as_int(x)));
    return x + __int_as_float(__builtin_amdgcn_ds_bpermute((lane ^ 32) << 2, __float_as_int(x)));
}

struct WinStride {
    int64_t b, l, h;
};
struct WinArgs {
    const void *q, *k, *v, *out, *gout;
    WinStride qs, ks, vs;      // elements; out and gout are contiguous [B, L, Hq, D]
    int B, L, Hq, Hkv, D, W, S;
    int tiles, ktiles;         // workgroups along the sequence: 64 queries, 32 keys each
    float scale;
    const int32_t *begin, *end;
    int mode, modeg;           // how rows of q, k, v / of out, gout are read
    int wide;                  // rows of out, dq take stores of four elements
    float *lse;                // [B, Hq, L]
    float *delta, *ref, *norm; // [B, Hq, L]: -delta; p 2^p_bits = exp2((s - ref) c - norm), see win_dq_kernel
    float* gmax;               // fp16: largest |dS| (before the scale) of every 16 queries [B, Hq, 4 tiles]
    float* part;               // far sinks: [B, Hkv, chunks, 2, S, D]
    int chunks;                // far sinks: workgroups along the sequence; 0: none
    int here;                  // far sinks: taken by win_dkdv_kernel itself
};
// [begin[b], end[b]) cut to the row, whatever the arrays hold
__device__ __forceinline__ void history(const int32_t* begin, const int32_t* end, int b, int L, int& lo, int& hi) {
    lo = begin ? begin[b] : 0;
    hi = end ? end[b] : L;
    lo = lo < 0 ? 0 : (lo > L ? L : lo);
    hi = hi < 0 ? 0 : (hi > L ? L : hi);
}
__device__ __forceinline__ void win_range(const WinArgs& a, int b, int& lo, int& hi) {
    history(a.begin, a.end, b, a.L, lo, hi);
}
// the keys a query sees through the window are [first, first + count); count 0: none
__device__ __forceinline__ void win_span(const WinArgs& a, int q, bool ok, int lo, int& first, int& count) {
    first = q - a.W + 1 > lo ? q - a.W + 1 : lo;
    count = ok ? q - first + 1 : 0;
}

// ---- staging of an R-row tile by 256 threads: rows t0 .. t0 + R - 1 of the sequence, those outside [lo, hi) as zeros ----
// A thread's places in the tile stay the same, so their offsets are worked out once and a tile inside [lo, hi) costs one
// 64-bit add per piece; only tiles at the ends clamp rows and clear what does not exist.
template <class T, int DP, int R, bool FAST>
struct Stage {
    static constexpr int OCTS = R * DP / 8, N = (OCTS + 255) / 256, LD = lds_ld<T, DP>();
    const T* base;
    int64_t ld, off[N];
    int lo, hi, D, mode, t0;
    Oct<T> r[N];
    __device__ __forceinline__ static int place(int n) {
        const int o = (int)threadIdx.x + n * 256;
        return OCTS % 256 == 0 || o < OCTS ? o : OCTS - 1;
    }
    __device__ __forceinline__ static int row(int n) { return place(n) / (DP / 8); }
    __device__ __forceinline__ static int col(int n) { return place(n) % (DP / 8) * 8; }
    __device__ __forceinline__ void init(const T* base_, int64_t ld_, int lo_, int hi_, int D_, int mode_) {
        base = base_;
        ld = ld_;
        lo = lo_;
        hi = hi_;
        D = D_;
        mode = mode_;
        t0 = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) off[n] = row(n) * ld + (col(n) < D ? col(n) : 0);
    }
    __device__ __forceinline__ bool inside() const { return t0 >= lo && t0 + R <= hi; }
    template <int MODE>
    __device__ __forceinline__ void load_edge() {
#pragma unroll
        for (int n = 0; n < N; ++n) r[n] = load_oct<T>(base + (int64_t)clamp_row(t0 + row(n), lo, hi) * ld, col(n), D, MODE);
    }
    __device__ __forceinline__ void load(int t) {
        t0 = t;
        if (FAST && inside()) {
            const T* p = base + (int64_t)t0 * ld;
#pragma unroll
            for (int n = 0; n < N; ++n) r[n] = load_oct<T>(p + off[n], 0, 8, WA_PIECES);
        } else if (FAST || mode == WA_PIECES) {                // one branch around all loads, not one around each
            load_edge<WA_PIECES>();
        } else if (mode == WA_WORDS) {
            load_edge<WA_WORDS>();
        } else {
            load_edge<WA_ELEMS>();
        }
    }
    __device__ __forceinline__ void store(T* tile) const {
        if (FAST && inside()) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (OCTS % 256 == 0 || (int)threadIdx.x + n * 256 < OCTS) lds_store_oct<T>(tile + row(n) * LD + col(n), r[n]);
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = t0 + row(n);
            const Oct<T> x = keep_oct<T>(r[n], at >= lo && at < hi ? D - col(n) : 0, FAST ? WA_PIECES : mode);
            if (OCTS % 256 == 0 || (int)threadIdx.x + n * 256 < OCTS) lds_store_oct<T>(tile + row(n) * LD + col(n), x);
        }
    }
};
// the row fragments of 16 rows (lane & 15) straight from memory; row: one that exists
template <class T, int DP, bool FAST>
__device__ __forceinline__ void load_frags(Oct<T> (&f)[DP / 32], const T* row, bool ok, int D, int mode) {
    const int g = (threadIdx.x & 63) >> 4;
    if (FAST) {
        D = DP;
        mode = WA_PIECES;
    }
    if (mode == WA_PIECES) {
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) f[s] = load_oct<T>(row, 32 * s + 8 * g, D, WA_PIECES);
    } else if (mode == WA_WORDS) {
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) f[s] = load_oct<T>(row, 32 * s + 8 * g, D, WA_WORDS);
    } else {
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) f[s] = load_oct<T>(row, 32 * s + 8 * g, D, WA_ELEMS);
    }
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) f[s] = keep_oct<T>(f[s], ok ? D - 32 * s - 8 * g : 0, mode);
}
// a 32-row tile staged by one wavefront, eight pieces of it in flight
template <class T, int DP, bool FAST, class Row>
__device__ __forceinline__ void wave_stage_rows(T* tile, const T* base, int D, int mode, Row row) {
    if (FAST) {
        D = DP;
        mode = WA_PIECES;
    }
    constexpr int LD = lds_ld<T, DP>(), N = WA_BK * DP / 8 / 64, STEP = N < 8 ? N : 8;
    const int lane = threadIdx.x & 63;
    auto part = [&](int n0, auto how) {
        Oct<T> r[STEP];
#pragma unroll
        for (int n = 0; n < STEP; ++n) {
            const int o = lane + (n0 + n) * 64;
            bool ok;
            r[n] = load_oct<T>(base + row(o / (DP / 8), ok), o % (DP / 8) * 8, D, decltype(how)::value);
        }
#pragma unroll
        for (int n = 0; n < STEP; ++n) {
            const int o = lane + (n0 + n) * 64, c = o % (DP / 8) * 8;
            bool ok;
            row(o / (DP / 8), ok);
            lds_store_oct<T>(tile + o / (DP / 8) * LD + c, keep_oct<T>(r[n], ok ? D - c : 0, decltype(how)::value));
        }
    };
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += STEP) {
        if (mode == WA_PIECES)
            part(n0, std::integral_constant<int, WA_PIECES>());
        else if (mode == WA_WORDS)
            part(n0, std::integral_constant<int, WA_WORDS>());
        else
            part(n0, std::integral_constant<int, WA_ELEMS>());
    }
}
template <class T, int DP, bool FAST>
__device__ __forceinline__ void wave_stage(T* tile, const T* base, int64_t ld, int row0, int lo, int hi, int D, int mode) {
    wave_stage_rows<T, DP, FAST>(tile, base, D, mode, [&](int r, bool& ok) {
        ok = row0 + r >= lo && row0 + r < hi;
        return (int64_t)clamp_row(row0 + r, lo, hi) * ld;
    });
}
// Workgroups go to the 8 XCDs in turn and each XCD has its own L2: dealt out one by one, neighbours along the sequence, which
// read the same rows, would fetch them into 8 caches.  So runs of WA_RUN neighbours go to one XCD, the runs in turn (whole
// eighths of the grid would leave an XCD with nothing but the short histories of a batch).  dK / dV of 4 x 2047 x 8 / 2 heads x
// 128 bf16 (P in one half): 56.5 us one by one, 54.0 in runs of 16, 53.6 in runs of 32; of 64 x 200 x 2 x 64 fp32: 35.3, 33.1, 32.6 us.
constexpr int WA_RUN = 32;
__device__ __forceinline__ unsigned win_block() {
    constexpr unsigned ROUND = 8 * WA_RUN;
    const unsigned id = blockIdx.x, base = id / ROUND * ROUND;
    if (base + ROUND > gridDim.x) return id;                   // what is left of the grid: as it comes
    return base + (id % 8) * WA_RUN + id % ROUND / 8;
}
// which key tiles a block of queries [qlo, qhi] needs: the tiles of the first items, then those of the window
struct KeyTiles {
    int s0, ns, w0, n;
    __device__ __forceinline__ void set(const WinArgs& a, int qlo, int qhi, int lo) {
        ns = n = 0;
        s0 = w0 = 0;
        if (qlo > qhi) return;
        const int first = qlo - a.W + 1 > lo ? qlo - a.W + 1 : lo;      // W <= L: no overflow
        w0 = first / WA_BK;
        if (a.S > 0) {
            s0 = lo / WA_BK;
            int s1 = (lo + a.S - 1) / WA_BK;
            if (s1 >= w0) s1 = w0 - 1;
            ns = s1 >= s0 ? s1 - s0 + 1 : 0;
        }
        n = ns + qhi / WA_BK - w0 + 1;
    }
    __device__ __forceinline__ int row0(int i) const { return (i < ns ? s0 + i : w0 + i - ns) * WA_BK; }
};

// ---- forward ---------------------------------------------------------------------------------------------------------------
// A workgroup of 4 wavefronts takes 64 queries of one head; the key and value tiles it needs go through LDS, the next
// tile's loads in flight while one is used (two buffers; one where two would not leave room for a second workgroup).
// NH = 2: two heads of a group at once, which share the tiles, the key and value operands read from LDS and the masks.
// 4 x 2047 x 8 / 2 heads x 128 bf16, window 256: 30.5 us, 8.0 useful GFLOP = 262 TFLOP/s.  LDS reads (16 KB a wavefront and
// tile), exponentials and matrix instructions take about a third each and overlap only across wavefronts (with P in one half,
// 28 us: 24.6 without its loads from memory, 19.4 without its products).  64 x 200 x 2 x 64 fp32, window 50: 18 us.
// Tried: 64 keys in one buffer instead of 32 in two, 35.6 us against 29.6.
template <class T, int DP>
constexpr int fwd_buffers() {
    return DP * (int)sizeof(T) <= 512 ? 2 : 1;
}
// Naming the workgroups per CU keeps the accumulators in ordinary registers: left alone the compiler moves all of them to
// the accumulation registers and back around every tile's rescaling (64 of 350 instructions).
template <class T, int DP, bool FAST, int NH>
__global__ __launch_bounds__(256, NH == 1 && DP * (int)sizeof(T) <= 256 ? 3 : (DP * (int)sizeof(T) <= 512 ? 2 : 1)) void win_fwd_kernel(WinArgs a, T* __restrict__ out, float* __restrict__ lse) {
    constexpr int LD = lds_ld<T, DP>(), NB = fwd_buffers<T, DP>(), TILE = WA_BK * LD;
    extern __shared__ char smem[];
    T* kt = reinterpret_cast<T*>(smem);
    T* vt = kt + NB * TILE;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const unsigned id = win_block();
    const int q0 = (int)(id % a.tiles) * 64, h = (int)(id / a.tiles % (a.Hq / NH)) * NH;   // this head, .. h + NH - 1
    const int b = (int)(id / a.tiles / (a.Hq / NH)), hk = h / (a.Hq / a.Hkv);
    int lo, hi;
    win_range(a, b, lo, hi);
    const T* kp = (const T*)a.k + b * a.ks.b + hk * a.ks.h;
    const T* vp = (const T*)a.v + b * a.vs.b + hk * a.vs.h;
    const int qw = q0 + wave * 16, qi = qw + c16;
    const bool q_ok = qi >= lo && qi < hi;
    const int qlo = qw > lo ? qw : lo, qhi = qw + 15 < hi - 1 ? qw + 15 : hi - 1;      // this wavefront's queries
    int k_first, k_count;
    win_span(a, qi, q_ok, lo, k_first, k_count);
    KeyTiles kts;
    kts.set(a, q0 > lo ? q0 : lo, q0 + 63 < hi - 1 ? q0 + 63 : hi - 1, lo);
    Stage<T, DP, WA_BK, FAST> ks, vs;
    ks.init(kp, a.ks.l, lo, hi, a.D, a.mode);
    vs.init(vp, a.vs.l, lo, hi, a.D, a.mode);
    if (kts.n > 0) {                                           // the first tile and the queries arrive together
        ks.load(kts.row0(0));
        vs.load(kts.row0(0));
    }
    Oct<T> qf[NH][DP / 32];
    f32x4 o[NH][DP / 16];
    float m[NH], l[NH];
#pragma unroll
    for (int y = 0; y < NH; ++y) {
        load_frags<T, DP, FAST>(qf[y], (const T*)a.q + b * a.qs.b + (int64_t)clamp_row(qi, lo, hi) * a.qs.l + (h + y) * a.qs.h, q_ok, a.D, a.mode);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[y][t] = f32x4{0, 0, 0, 0};
        m[y] = -__builtin_inff();
        l[y] = 0.0f;
    }
    const float c = a.scale * WA_LOG2E;
    if (kts.n > 0) {
        ks.store(kt);
        vs.store(vt);
    }
    __syncthreads();
    for (int n = 0; n < kts.n; ++n) {
        const int t0 = kts.row0(n);
        const T* kc = kt + (NB == 2 ? (n & 1) * TILE : 0);
        const T* vc = vt + (NB == 2 ? (n & 1) * TILE : 0);
        if (n + 1 < kts.n) {
            ks.load(kts.row0(n + 1));
            vs.load(kts.row0(n + 1));
        }
        if (qlo <= qhi && t0 <= qhi && (t0 + WA_BK - 1 > qlo - a.W || t0 < lo + a.S)) {
            f32x4 s[NH][2];
#pragma unroll
            for (int y = 0; y < NH; ++y) s[y][0] = s[y][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < DP / 32; ++x) {
                const Oct<T> k0 = row_frag<T>(kc + c16 * LD + 32 * x + 8 * g), k1 = row_frag<T>(kc + (16 + c16) * LD + 32 * x + 8 * g);
#pragma unroll
                for (int y = 0; y < NH; ++y) {
                    s[y][0] = mma(k0, qf[y][x], s[y][0]);
                    s[y][1] = mma(k1, qf[y][x], s[y][1]);
                }
            }
            // a tile that all 16 queries see whole needs no mask
            const bool whole = t0 >= lo && t0 + WA_BK - 1 <= qw && qw >= lo && qw + 15 < hi && qw + 15 - t0 < a.W;
            if (!whole) {
                const int k0 = t0 + 4 * g;
                if (t0 < lo + a.S) {                           // the tile holds first items
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int k = k0 + 16 * x + i;
                            const bool first = ((unsigned)(k - lo) < (unsigned)a.S) & (k <= qi) & q_ok;
                            const bool seen = ((unsigned)(k - k_first) < (unsigned)k_count) | first;
#pragma unroll
                            for (int y = 0; y < NH; ++y) s[y][x][i] = seen ? s[y][x][i] : -__builtin_inff();
                        }
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool seen = (unsigned)(k0 + 16 * x + i - k_first) < (unsigned)k_count;
#pragma unroll
                            for (int y = 0; y < NH; ++y) s[y][x][i] = seen ? s[y][x][i] : -__builtin_inff();
                        }
                }
            }
            Oct<T> p[NH], pl[NH];                              // 16-bit types: the halves of P
#pragma unroll
            for (int y = 0; y < NH; ++y) {
                float mt = s[y][0][0];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[y][x][i]);
                mt = groups_max(mt);
                // m: the largest score itself.  Its weight is 2^0 whatever the scores' size: with m c rounded, and s c - m c
                // in one fma, it would be 2 to the rounding error of m c, beyond any range from scores of 2^31 on
                const float mn = fmaxf(m[y], mt), ms = mn == -__builtin_inff() ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f((m[y] - ms) * c);
                m[y] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[y][x][i] = weight<T>(s[y][x][i] - ms, c);
                        sum += s[y][x][i];
                    }
                l[y] = fmaf(l[y], alpha, sum);
                if (__ballot(alpha != 1.0f) != 0) {
#pragma unroll
                    for (int t = 0; t < DP / 16; ++t) o[y][t] *= alpha;
                }
                if constexpr (sizeof(T) == 2)
                    split_oct<T>(s[y][0], s[y][1], p[y], pl[y]);
                else
                    p[y] = to_oct<T>(s[y][0], s[y][1]);
            }
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                const Oct<T> vf = col_frag<T, LD>(vc, 16 * t);
#pragma unroll
                for (int y = 0; y < NH; ++y) {
                    o[y][t] = mma(vf, p[y], o[y][t]);
                    if constexpr (sizeof(T) == 2) o[y][t] = mma(vf, pl[y], o[y][t]);
                }
            }
        }
        if (NB == 1) __syncthreads();
        if (n + 1 < kts.n) {
            ks.store(kt + (NB == 2 ? ((n + 1) & 1) * TILE : 0));
            vs.store(vt + (NB == 2 ? ((n + 1) & 1) * TILE : 0));
        }
        __syncthreads();
    }
#pragma unroll
    for (int y = 0; y < NH; ++y) l[y] = groups_sum(l[y]);
    if (qi >= a.L) return;
#pragma unroll
    for (int y = 0; y < NH; ++y) {
        const float inv = l[y] == 0.0f ? 0.0f : 1.0f / l[y];                   // a NaN stays one
        T* op = out + (((int64_t)b * a.L + qi) * a.Hq + h + y) * a.D;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            const int d = 16 * t + 4 * g;
            if (FAST || (d + 4 <= a.D && a.wide)) {
                float r[4] = {o[y][t][0] * inv, o[y][t][1] * inv, o[y][t][2] * inv, o[y][t][3] * inv};
                store_f32<T, 4>(op + d, r);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < a.D) op[d + i] = (T)(o[y][t][i] * inv);
            }
        }
        if (g == 0) lse[((int64_t)b * a.Hq + h + y) * a.L + qi] = l[y] == 0.0f ? -__builtin_inff() : fmaf(m[y], a.scale, (log2f(l[y]) - p_bits<T>()) * WA_LN2);
    }
}

// ---- backward: dQ ------------------------------------------------------------------------------------------------------------
// dS = P (dP - delta) scale with delta_i = sum_j p_ij dP_ij;  dQ^T = K^T dS^T in the forward's layout.  Writes delta for the
// others.  dP - delta cancels where one key carries a row, so delta has to be as exact as dP.  For fp32 it is <dO_i, O_i>;
// a 16-bit O is off by half a step (uncorrected, dQ and dK were 1.8 times as far from 64 bits as the rounding of the result
// alone).  16-bit types start from that delta_0 and correct it: with r = sum p (dP - delta_0) = delta - delta_0,
//   dQ = scale (sum p (dP - delta_0) K - r sum p K),
// r being small, the second sum needs no more than P rounded to 16 bits.  The first one's weights are split into two halves
// (hi + what hi misses), one more matrix instruction instead of another half step lost.  (Running the tiles twice, first
// for delta, is as exact and took 77 us where this took 48 at 4 x 2047 x 8 x 128.)
// P from lse alone would be off by lse's rounding: 1e-3 of P at scores of 1e4.  So lse only gives a reference near the row's
// maximum, ref = lse / scale; the kernel, which sees the whole row, sums the weights 2^((s - ref) c) itself, divides by the sum
// l in the end and hands ref and norm = log2 l to the others.  Where |lse| reaches WA_FAR its rounding (half a unit of log 2 at
// 2^23) could carry the weights out of range: there the workgroup takes the maximum itself in a first run over the keys
// (backward of 4 x 2047 x 8 / 2 x 128 bf16: 137 us, 121 without).
constexpr float WA_FAR = 65536.0f;
// fp16 holds dS of no gradient, value or scale by itself: it is multiplied by a power of two that brings the largest |dS| to
// [2^13, 2^14), so that nothing overflows and the two halves keep 2^-38 of the largest.  Here that power, at most 2^100
// (dS = 0); 1 for what is not finite.
__device__ __forceinline__ float grad_up(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 255u);
    return e == 255 ? 1.0f : __uint_as_float((uint32_t)(e > 40 ? 267 - e : 227) << 23);
}
template <class T, int DP, bool FAST>
__global__ __launch_bounds__(256, DP * (int)sizeof(T) <= 256 ? 2 : 1) void win_dq_kernel(WinArgs a, T* __restrict__ dq) {
    constexpr int LD = lds_ld<T, DP>(), NB = fwd_buffers<T, DP>(), TILE = WA_BK * LD;
    constexpr bool FIX = sizeof(T) == 2;                                     // delta is corrected
    extern __shared__ char smem[];
    T* kt = reinterpret_cast<T*>(smem);
    T* vt = kt + NB * TILE;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const unsigned id = win_block();
    const int q0 = (int)(id % a.tiles) * 64, h = (int)(id / a.tiles % a.Hq);
    const int b = (int)(id / a.tiles / a.Hq), hk = h / (a.Hq / a.Hkv);
    int lo, hi;
    win_range(a, b, lo, hi);
    const T* kp = (const T*)a.k + b * a.ks.b + hk * a.ks.h;
    const T* vp = (const T*)a.v + b * a.vs.b + hk * a.vs.h;
    const int qw = q0 + wave * 16, qi = qw + c16, qc = clamp_row(qi, lo, hi);
    const bool q_ok = qi >= lo && qi < hi;
    const int qlo = qw > lo ? qw : lo, qhi = qw + 15 < hi - 1 ? qw + 15 : hi - 1;
    int k_first, k_count;
    win_span(a, qi, q_ok, lo, k_first, k_count);
    KeyTiles kts;
    kts.set(a, q0 > lo ? q0 : lo, q0 + 63 < hi - 1 ? q0 + 63 : hi - 1, lo);
    Stage<T, DP, WA_BK, FAST> ks, vs;
    ks.init(kp, a.ks.l, lo, hi, a.D, a.mode);
    vs.init(vp, a.vs.l, lo, hi, a.D, a.mode);
    if (kts.n > 0) {
        ks.load(kts.row0(0));
        vs.load(kts.row0(0));
    }
    Oct<T> qf[DP / 32], gf[DP / 32];
    const int64_t irow = (((int64_t)b * a.L + qc) * a.Hq + h) * a.D, srow = ((int64_t)b * a.Hq + h) * a.L;
    load_frags<T, DP, FAST>(qf, (const T*)a.q + b * a.qs.b + (int64_t)qc * a.qs.l + h * a.qs.h, q_ok, a.D, a.mode);
    load_frags<T, DP, FAST>(gf, (const T*)a.gout + irow, q_ok, a.D, a.modeg);
    float ref = q_ok ? a.lse[srow + qc] / a.scale : 0.0f, l = 0.0f;
    bool far;                                                                // the same in all four wavefronts
    {
        const int at = q0 + lane;
        const float x = at >= lo && at < hi ? a.lse[srow + at] : 0.0f;
        far = __ballot(!(fabsf(x) < WA_FAR)) != 0;
    }
    float delta = 0.0f, fix = 0.0f;
    {
        Oct<T> of[DP / 32];
        load_frags<T, DP, FAST>(of, (const T*)a.out + irow, q_ok, a.D, a.modeg);
#pragma unroll
        for (int s = 0; s < DP / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], (float)of[s][e], delta);
        delta = groups_sum(delta);
    }
    // fp16: the power of two starts from a guess (|dP| of about 8 |dO|) and follows the query's largest |dS| down as the tiles
    // come, as the forward's maximum goes up: no |dS| up beyond 2^15
    constexpr bool RANGE = std::is_same<T, f16>::value;
    float up = 1.0f, most = 0.0f, big = 0.0f;
    if constexpr (RANGE) {
        float x = 0.0f;
#pragma unroll
        for (int s = 0; s < DP / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) x = fmaxf(x, fabsf((float)gf[s][e]));
        up = grad_up(8.0f / p_down<T>() * groups_max(x));
        most = 32768.0f / up;
    }
    f32x4 acc[DP / 16], pk[FIX ? DP / 16 : 1];                               // sums of p (dP - delta) K and of p K
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        acc[t] = f32x4{0, 0, 0, 0};
        if (FIX) pk[t] = f32x4{0, 0, 0, 0};
    }
    const float c = a.scale * WA_LOG2E;
    // whether this wavefront's queries see anything of the tile
    auto needs = [&](int t0) { return qlo <= qhi && t0 <= qhi && (t0 + WA_BK - 1 > qlo - a.W || t0 < lo + a.S); };
    auto sees = [&](int k) {
        return ((unsigned)(k - k_first) < (unsigned)k_count) | (((unsigned)(k - lo) < (unsigned)a.S) & (k <= qi) & q_ok);
    };
    if (far) {
        float mx = -__builtin_inff();
        for (int n = 0; n < kts.n; ++n) {
            const int t0 = kts.row0(n);
            ks.load(t0);
            __syncthreads();
            ks.store(kt);
            __syncthreads();
            if (!needs(t0)) continue;
            f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int x = 0; x < DP / 32; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) s[y] = mma(row_frag<T>(kt + (16 * y + c16) * LD + 32 * x + 8 * g), qf[x], s[y]);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sees(t0 + 16 * y + 4 * g + i) ? s[y][i] : -__builtin_inff());
        }
        mx = groups_max(mx);
        ref = mx == -__builtin_inff() ? 0.0f : mx;
        if (kts.n > 0) ks.load(kts.row0(0));                                 // the values' first tile is still held
        __syncthreads();
    }
    if (kts.n > 0) {
        ks.store(kt);
        vs.store(vt);
    }
    __syncthreads();
    for (int n = 0; n < kts.n; ++n) {
        const int t0 = kts.row0(n);
        const T* kc = kt + (NB == 2 ? (n & 1) * TILE : 0);
        const T* vc = vt + (NB == 2 ? (n & 1) * TILE : 0);
        if (n + 1 < kts.n) {
            ks.load(kts.row0(n + 1));
            vs.load(kts.row0(n + 1));
        }
        if (needs(t0)) {
            f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
            f32x4 dp[2] = {f32x4{-delta, -delta, -delta, -delta}, f32x4{-delta, -delta, -delta, -delta}};   // dP - delta
#pragma unroll
            for (int x = 0; x < DP / 32; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    s[y] = mma(row_frag<T>(kc + (16 * y + c16) * LD + 32 * x + 8 * g), qf[x], s[y]);
                    dp[y] = mma(row_frag<T>(vc + (16 * y + c16) * LD + 32 * x + 8 * g), gf[x], dp[y]);
                }
            const bool whole = t0 >= lo && t0 + WA_BK - 1 <= qw && qw >= lo && qw + 15 < hi && qw + 15 - t0 < a.W;
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[y][i] = weight<T>(s[y][i] - ref, c);
            if (!whole) {
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = sees(t0 + 16 * y + 4 * g + i);
                        s[y][i] = seen ? s[y][i] : 0.0f;
                        dp[y][i] = seen ? dp[y][i] : 0.0f;     // whatever it was: 0 times a finite number
                    }
            }
            const Oct<T> p = to_oct<T>(s[0], s[1]);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    l += s[y][i];
                    s[y][i] *= dp[y][i];
                    fix += s[y][i];
                }
            if constexpr (RANGE) {
                float t = 0.0f;
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) t = fmaxf(t, fabsf(s[y][i]));
                big = fmaxf(big, t);
                if (__ballot(t > most) != 0) {
                    t = groups_max(t);
                    const float next = t > most ? grad_up(t) : up, f = next / up;
                    up = next;
                    most = 32768.0f / up;
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) acc[x] *= f;
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) s[y] *= up;
            }
            if constexpr (FIX) {
                Oct<T> dh, dl;
                split_oct<T>(s[0], s[1], dh, dl);
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) {
                    const Oct<T> kf = col_frag<T, LD>(kc, 16 * t);
                    acc[t] = mma(kf, dh, acc[t]);
                    pk[t] = mma(kf, p, pk[t]);
                    acc[t] = mma(kf, dl, acc[t]);
                }
            } else {
                const Oct<T> ds = to_oct<T>(s[0], s[1]);
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) acc[t] = mma(col_frag<T, LD>(kc, 16 * t), ds, acc[t]);
            }
        }
        if (NB == 1) __syncthreads();
        if (n + 1 < kts.n) {
            ks.store(kt + (NB == 2 ? ((n + 1) & 1) * TILE : 0));
            vs.store(vt + (NB == 2 ? ((n + 1) & 1) * TILE : 0));
        }
        __syncthreads();
    }
    l = groups_sum(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;                           // a NaN stays one
    if constexpr (FIX) {
        fix = groups_sum(fix) * inv;
        delta += fix;
        const float f = -fix * up;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(f, pk[t][i], acc[t][i]);
    }
    if constexpr (RANGE) {
        // no |dS| of these 16 queries is larger: p (dP - delta) = p (dP - delta_0) - p fix
        big = groups_max(big) * inv + fabsf(fix);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor(big, off, 64));
        if (lane == 0) a.gmax[(((int64_t)b * a.Hq + h) * a.tiles + q0 / 64) * 4 + wave] = big;
    }
    if (qi >= a.L) return;
    if (g == 0) {
        a.delta[srow + qi] = -delta;
        a.ref[srow + qi] = ref;
        a.norm[srow + qi] = l == 0.0f ? 0.0f : log2f(l * p_down<T>()) - p_bits<T>();
    }
    const float down = inv * a.scale / up;
    T* op = dq + (((int64_t)b * a.L + qi) * a.Hq + h) * a.D;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const int d = 16 * t + 4 * g;
        if (FAST || (d + 4 <= a.D && a.wide)) {
            float r[4] = {acc[t][0] * down, acc[t][1] * down, acc[t][2] * down, acc[t][3] * down};
            store_f32<T, 4>(op + d, r);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d + i < a.D) op[d + i] = (T)(acc[t][i] * down);
        }
    }
}

// ---- backward: dK, dV --------------------------------------------------------------------------------------------------------
// S = Q K^T here, so a lane holds one KEY and four queries of each 16: the A operand of dV = P^T dO and dK = dS^T Q.
// 4 x 2047 x 8 / 2 heads x 128 bf16, window 256: 58 us (dQ: 51 us), 64 x 200 x 2 x 64 fp32: 33 us (26 us).  A step of 32 queries
// x 16 keys reads 33 KB from LDS for 48 matrix instructions: LDS takes half of the time, and 32 keys a wavefront, which
// would halve that, do not fit the registers at D = 128.
// one (32 queries x 16 keys) step: adds to dk, dv what the queries [q_first, q_first + q_count) give the lane's key (whole:
// all of them do)
template <class T, int DP>
__device__ __forceinline__ void dkdv_step(const WinArgs& a, const T* qc, const T* gc, const float* ref, const float* norm, const float* delta,
                                          const Oct<T> (&kf)[DP / 32], const Oct<T> (&vf)[DP / 32], int t0, int q_first,
                                          int q_count, bool whole, float up, f32x4 (&dk)[DP / 16],
                                          f32x4 (&dv)[DP / 16]) {
    constexpr int LD = lds_ld<T, DP>();
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const float c = a.scale * WA_LOG2E;
    f32x4 s[2], dp[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        s[y] = f32x4{0, 0, 0, 0};
        dp[y] = *reinterpret_cast<const f32x4*>(delta + 16 * y + 4 * g);     // -delta: the sum becomes dP - delta
    }
#pragma unroll
    for (int x = 0; x < DP / 32; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            s[y] = mma(row_frag<T>(qc + (16 * y + c16) * LD + 32 * x + 8 * g), kf[x], s[y]);
            dp[y] = mma(row_frag<T>(gc + (16 * y + c16) * LD + 32 * x + 8 * g), vf[x], dp[y]);
        }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const f32x4 rf = *reinterpret_cast<const f32x4*>(ref + 16 * y + 4 * g);
        const f32x4 nm = *reinterpret_cast<const f32x4*>(norm + 16 * y + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p = __builtin_amdgcn_exp2f(fmaf(s[y][i] - rf[i], c, -nm[i])), d = dp[y][i];
            if (!whole && (unsigned)(t0 + 16 * y + 4 * g + i - q_first) >= (unsigned)q_count) p = d = 0.0f;
            s[y][i] = p;
            dp[y][i] = p * d * up;                               // in this order: only p d is known to be in range
        }
    }
    if constexpr (sizeof(T) == 2) {
        Oct<T> ph, pl, dh, dl;
        split_oct<T>(s[0], s[1], ph, pl);
        split_oct<T>(dp[0], dp[1], dh, dl);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            const Oct<T> gf = col_frag<T, LD>(gc, 16 * t);
            dv[t] = mma(ph, gf, dv[t]);
            dv[t] = mma(pl, gf, dv[t]);
            const Oct<T> qf = col_frag<T, LD>(qc, 16 * t);
            dk[t] = mma(dh, qf, dk[t]);
            dk[t] = mma(dl, qf, dk[t]);
        }
    } else {
        const Oct<T> pf = to_oct<T>(s[0], s[1]), df = to_oct<T>(dp[0], dp[1]);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            dv[t] = mma(pf, col_frag<T, LD>(gc, 16 * t), dv[t]);
            dk[t] = mma(df, col_frag<T, LD>(qc, 16 * t), dk[t]);
        }
    }
}

// The power of two for dS of the queries [q0, q1] of a group's heads (fp16: grad_up of the largest |dS| that win_dq_kernel met;
// queries whose dS is not finite give what they see no finite gradient, whatever it is)
// In two steps, with loads of the caller's own between them: first() requests a lane's first value, scale() the rest and
// gives the answer.
template <class T>
struct GradScale {
    const float* rows;                                       // [heads, 4 tiles] of the group
    int r0, n, total, tiles;
    float x;
    __device__ __forceinline__ float at(int i) const { return rows[(int64_t)(i / n) * tiles * 4 + r0 + i % n]; }
    __device__ __forceinline__ void first(const WinArgs& a, int b, int h0, int heads, int q0, int q1) {
        if constexpr (!std::is_same<T, f16>::value) return;
        rows = a.gmax + ((int64_t)b * a.Hq + h0) * a.tiles * 4;
        tiles = a.tiles;
        r0 = q0 / 16;
        n = q1 / 16 - r0 + 1;
        total = n * heads;
        const int i = threadIdx.x & 63;
        x = at(i < total ? i : 0);
    }
    __device__ __forceinline__ float scale() const {
        if constexpr (!std::is_same<T, f16>::value) return 1.0f;
        float big = x < __builtin_inff() ? x : 0.0f;
        for (int i = (int)(threadIdx.x & 63) + 64; i < total; i += 64) {
            const float y = at(i);
            big = fmaxf(big, y < __builtin_inff() ? y : 0.0f);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor(big, off, 64));
        return grad_up(big);
    }
};
// A workgroup takes 32 keys of one key head and walks the queries that see them through the window, 64 at a time, head by
// head of the group (so the group's sum needs no atomics): wavefront (w, x) takes key half w and query half x, the halves
// of the queries are added up at the end.  What the first items get from queries beyond the window is found here too
// where that is at most 8 more steps (backward of 64 x 200 x 2 x 64 fp32 with 2 first items, 3 steps: 62 us, 65 us with a launch
// of its own; 32 x 600, 9 steps: 101 and 93 us); else it comes from win_sink_kernel's partial sums, added last and in order.
// (One buffer: with two the two workgroups on the CU, which hide each other's barriers, gain nothing.)
// a second workgroup on the CU is worth more than registers to spare (at D <= 128 in 16 bits, 64 in fp32)
template <class T, int DP, bool FAST>
__global__ __launch_bounds__(256, DP * (int)sizeof(T) <= 256 ? 2 : 1) void win_dkdv_kernel(WinArgs a, T* __restrict__ dk_out, T* __restrict__ dv_out) {
    constexpr int LD = lds_ld<T, DP>(), R = 64, TILE = R * LD;
    constexpr bool AHEAD = DP * (int)sizeof(T) <= 512;       // else the next tile does not fit the registers
    extern __shared__ char smem[];
    T* qt = reinterpret_cast<T*>(smem);
    T* gt = qt + TILE;
    float* st = reinterpret_cast<float*>(gt + TILE);         // [4][64]: ref, norm, -delta twice (a branch costs 3 us)
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const unsigned id = win_block();
    const int k0 = (int)(id % a.ktiles) * 32, hk = (int)(id / a.ktiles % a.Hkv);
    const int b = (int)(id / a.ktiles / a.Hkv), G = a.Hq / a.Hkv, half = (wave >> 1) * 32;
    int lo, hi;
    win_range(a, b, lo, hi);
    const int kw = k0 + (wave & 1) * 16, ki = kw + c16;
    const bool k_ok = ki >= lo && ki < hi;
    // the queries that see the key: [ki, ki + q_count), through the window or (first items, when they are taken here) all
    const int first_end = a.here ? lo + a.S : lo;            // keys below it are first items taken here
    const int q_count = k_ok ? (ki >= first_end && hi - ki > a.W ? a.W : hi - ki) : 0;
    const int klo = k0 > lo ? k0 : lo, khi = k0 + 31 < hi - 1 ? k0 + 31 : hi - 1;
    const int qend = klo > khi ? -1 : (klo >= first_end && khi + (int64_t)a.W - 1 < hi - 1 ? khi + a.W - 1 : hi - 1);
    const int tq0 = klo / 32 * 32, nt = klo <= khi ? (qend - tq0) / R + 1 : 0, total = nt * G;
    Stage<T, DP, R, FAST> qs, gs;
    qs.init((const T*)a.q + b * a.qs.b + hk * G * a.qs.h, a.qs.l, lo, hi, a.D, a.mode);
    gs.init((const T*)a.gout + ((int64_t)b * a.L * a.Hq + hk * G) * a.D, (int64_t)a.Hq * a.D, lo, hi, a.D, a.modeg);
    float stat = 0.0f;
    const float* stats = wave == 0 ? a.ref : wave == 1 ? a.norm : a.delta;
    int h_next = 0, i_next = 0;                              // next tile: head of the group, place along the sequence
    auto load = [&]() {
        const int t0 = tq0 + i_next * R;
        qs.load(t0);
        gs.load(t0);
        {
            const int qi = t0 + (int)(threadIdx.x & (R - 1));
            const int64_t row = ((int64_t)b * a.Hq + hk * G + h_next) * a.L + clamp_row(qi, lo, hi);
            stat = stats[row];
            if (qi < lo || qi >= hi) stat = 0.0f;
        }
        if (++i_next == nt) {
            i_next = 0;
            ++h_next;
            qs.base += a.qs.h;
            gs.base += a.D;
        }
    };
    auto store = [&]() {
        qs.store(qt);
        gs.store(gt);
        st[threadIdx.x] = stat;
    };
    GradScale<T> ds_up;
    if (total > 0) {
        ds_up.first(a, b, hk * G, G, tq0, qend);
        load();
    }
    Oct<T> kf[DP / 32], vf[DP / 32];
    load_frags<T, DP, FAST>(kf, (const T*)a.k + b * a.ks.b + (int64_t)clamp_row(ki, lo, hi) * a.ks.l + hk * a.ks.h, k_ok, a.D, a.mode);
    load_frags<T, DP, FAST>(vf, (const T*)a.v + b * a.vs.b + (int64_t)clamp_row(ki, lo, hi) * a.vs.l + hk * a.vs.h, k_ok, a.D, a.mode);
    f32x4 dk[DP / 16], dv[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) dk[t] = dv[t] = f32x4{0, 0, 0, 0};
    const float up = total > 0 ? ds_up.scale() : 1.0f;
    if (total > 0) store();
    __syncthreads();
    for (int n = 0, i = 0; n < total; ++n) {
        const int t0 = tq0 + i * R + half;
        if (++i == nt) i = 0;
        if (AHEAD && n + 1 < total) load();
        if (kw <= t0 + 31 && (t0 - (kw + 15) < a.W || kw < first_end) && t0 < hi && kw < hi && kw + 15 >= lo) {
            const bool whole = kw >= lo && kw + 15 <= t0 && t0 + 31 < hi && t0 + 31 - kw < a.W;
            dkdv_step<T, DP>(a, qt + half * LD, gt + half * LD, st + half, st + R + half, st + 2 * R + half, kf, vf, t0, ki, q_count, whole,
                             up * p_down<T>(), dk, dv);
        }
        __syncthreads();
        if (!AHEAD && n + 1 < total) load();
        if (n + 1 < total) store();
        __syncthreads();
    }
    // the second query half's sums join the first's over LDS: [key half][2][16][DP] fp32, which the tiles have room for.
    // dK gets its scale here, in fp32: before, it could carry dS out of fp16's range
    const float down = a.scale / up;
    float* red = reinterpret_cast<float*>(smem) + (wave & 1) * 32 * DP;
#pragma unroll
    for (int which = 0; which < 2; ++which)
        if (wave >= 2) {
#pragma unroll
            for (int t = 0; t < DP / 16; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    red[which * 16 * DP + (4 * g + i) * DP + 16 * t + c16] = which ? dv[t][i] * p_down<T>() : dk[t][i] * down;
        }
    __syncthreads();
    const int far = a.chunks > 0 && klo <= khi && k0 < lo + a.S ? (lo + a.S < khi + 1 ? lo + a.S : khi + 1) - klo : 0;
    if (far > 0) {                                           // workgroup-uniform: first items klo .. klo + far - 1
        const int64_t step = 2 * (int64_t)a.S * a.D;
        const float* p = a.part + ((int64_t)b * a.Hkv + hk) * a.chunks * step + (int64_t)(klo - lo) * a.D;
        for (int e = threadIdx.x; e < 2 * far * a.D; e += 256) {
            const int which = e / (far * a.D), r = e - which * far * a.D, key = klo - k0 + r / a.D, d = r % a.D;
            const float* pe = p + (int64_t)which * a.S * a.D + r;
            float x = 0.0f;
            for (int q0 = 0; q0 < a.chunks; q0 += 16) {      // 16 chunks requested together
                float v[16];
#pragma unroll
                for (int q = 0; q < 16; ++q) v[q] = pe[(q0 + q < a.chunks ? q0 + q : 0) * step];
#pragma unroll
                for (int q = 0; q < 16; ++q) x += q0 + q < a.chunks ? v[q] : 0.0f;
            }
            reinterpret_cast<float*>(smem)[(key >> 4) * 32 * DP + which * 16 * DP + (key & 15) * DP + d] += x;
        }
        __syncthreads();
    }
    if (wave >= 2) return;
    // lane: column d = 16 t + c16 of keys kw + 4 g + i
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kk = kw + 4 * g + i;
        if (kk >= a.L) continue;
        T* ko = dk_out + (((int64_t)b * a.L + kk) * a.Hkv + hk) * a.D;
        T* vo = dv_out + (((int64_t)b * a.L + kk) * a.Hkv + hk) * a.D;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            const int d = 16 * t + c16;
            if (!FAST && d >= a.D) continue;
            const float x = fmaf(dk[t][i], down, red[(4 * g + i) * DP + d]);
            const float y = fmaf(dv[t][i], p_down<T>(), red[16 * DP + (4 * g + i) * DP + d]);
            ko[d] = (T)x;
            vo[d] = (T)y;
        }
    }
}

// ---- backward: what the first items get from queries beyond the window ----------------------------------------------------------
// Every query of a long history sees them, so their sums are split over chunks of 64 queries: NW wavefronts, each with its
// own tiles of 32 queries in LDS, all on the same 16 first items, added up over LDS in order.  4 x 2047 x 8 / 2 heads x 128 bf16:
// 12 us, bound by the latency of a chunk's loads; every wavefront does one or two tiles.
constexpr int WA_CHUNK = 64;
template <class T, int DP>
constexpr int sink_waves() {
    return DP * (int)sizeof(T) <= 256 ? 4 : (DP * (int)sizeof(T) <= 512 ? 2 : 1);
}
template <class T, int DP, bool FAST>
__global__ __launch_bounds__(256) void win_sink_kernel(WinArgs a) {
    constexpr int LD = lds_ld<T, DP>(), TILE = WA_BK * LD, NW = sink_waves<T, DP>();
    extern __shared__ char smem[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    T* qt = reinterpret_cast<T*>(smem) + wave * 2 * TILE;
    T* gt = qt + TILE;
    float* st = reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + NW * 2 * TILE) + wave * 128;
    const int groups = (a.S + 15) / 16;
    int id = (int)blockIdx.x;
    const int grp = id % groups;
    id /= groups;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int hk = id % a.Hkv, b = id / a.Hkv, G = a.Hq / a.Hkv;
    int lo, hi;
    win_range(a, b, lo, hi);
    const int kw = lo + grp * 16, ki = kw + c16;
    const bool k_ok = ki < hi && ki - lo < a.S;
    const int q_count = k_ok && hi - ki > a.W ? hi - ki - a.W : 0;        // queries beyond the window: from ki + window on
    Oct<T> kf[DP / 32], vf[DP / 32];
    load_frags<T, DP, FAST>(kf, (const T*)a.k + b * a.ks.b + (int64_t)clamp_row(ki, lo, hi) * a.ks.l + hk * a.ks.h, k_ok, a.D, a.mode);
    load_frags<T, DP, FAST>(vf, (const T*)a.v + b * a.vs.b + (int64_t)clamp_row(ki, lo, hi) * a.vs.l + hk * a.vs.h, k_ok, a.D, a.mode);
    f32x4 dk[DP / 16], dv[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) dk[t] = dv[t] = f32x4{0, 0, 0, 0};
    const int first = chunk * WA_CHUNK, per = WA_CHUNK / WA_BK;
    GradScale<T> ds_up;
    ds_up.first(a, b, hk * G, G, first, first + WA_CHUNK <= a.L ? first + WA_CHUNK - 1 : a.L - 1);
    const float up = ds_up.scale();
    const float down = a.scale / up;
    for (int n = wave; n < per * G; n += NW) {
        const int h = hk * G + n / per, t0 = first + n % per * WA_BK;
        // wavefront-uniform: no query of the tile is both in the history and beyond the window of the group's first key
        if (t0 >= hi || t0 + WA_BK - 1 - kw < a.W) continue;
        const T* qp = (const T*)a.q + b * a.qs.b + h * a.qs.h;
        const T* gp = (const T*)a.gout + ((int64_t)b * a.L * a.Hq + h) * a.D;
        wave_stage<T, DP, FAST>(qt, qp, a.qs.l, t0, lo, hi, a.D, a.mode);
        wave_stage<T, DP, FAST>(gt, gp, (int64_t)a.Hq * a.D, t0, lo, hi, a.D, a.modeg);
        {
            const int qi = t0 + (lane & 31);
            const int64_t row = ((int64_t)b * a.Hq + h) * a.L + clamp_row(qi, lo, hi);
            const bool in = qi >= lo && qi < hi;
            const float x = (lane < 32 ? a.ref : a.norm)[row], y = a.delta[row];
            st[lane] = in ? x : 0.0f;
            st[64 + lane] = in ? y : 0.0f;                       // the upper half's copies are not read
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
        dkdv_step<T, DP>(a, qt, gt, st, st + 32, st + 64, kf, vf, t0, ki + a.W, q_count, false, up * p_down<T>(), dk, dv);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // the wavefronts' sums in order through LDS (the tiles are done with), then to this chunk's slot
    const int64_t step = 2 * (int64_t)a.S * a.D;
    float* part = a.part + (((int64_t)b * a.Hkv + hk) * a.chunks + chunk) * step;
    float* red = reinterpret_cast<float*>(smem);             // [16][DP]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        for (int w = 0; w < NW; ++w) {
            __syncthreads();
            if (wave == w) {
#pragma unroll
                for (int t = 0; t < DP / 16; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* r = red + (4 * g + i) * DP + 16 * t + c16;
                        const float x = which ? dv[t][i] * p_down<T>() : dk[t][i] * down;
                        *r = w == 0 ? x : *r + x;
                    }
            }
        }
        __syncthreads();
        for (int o = threadIdx.x; o < 16 * DP; o += NW * 64) {
            const int r = o / DP, d = o % DP;
            if (grp * 16 + r < a.S && d < a.D) part[(int64_t)which * a.S * a.D + (int64_t)(grp * 16 + r) * a.D + d] = red[o];
        }
    }
}

// ---- one new token per sequence over a cache -----------------------------------------------------------------------------------
// The query stands at position end - 1 and sees the first items and the window before it.  A workgroup takes one key head
// (its up to 16 query heads are the 16 columns of the tile) and a share of the visible keys; its wavefronts take 32 keys
// in turn, keys straight into registers, values through their own LDS tile, and are joined at the end.  With few sequences
// the keys are split over workgroups and win_join_kernel adds up.  64 x 260 keys x 8 / 2 heads x 64 bf16: 7 us, three round trips
// to memory one after the other (8 wavefronts or loads a tile ahead: 6.5 us); 64 x 4096 keys: 28 us = 4.8 TB/s;
// one sequence of 300000 keys: 36 us = 4.2 TB/s.
struct TokenArgs {
    const void *q, *k, *v;
    int64_t qb, qh;
    WinStride ks, vs;
    int B, L, Hq, Hkv, D, W, S, splits, per, hgroups;   // per: 32-key tiles of a workgroup
    float scale;
    const int32_t *begin, *end;
    int mode, modeq;
    void* out;                                          // [B, Hq, D]
    float* part;                                        // [B, Hq, splits, D + 2]: sum, m, l
};
template <class T, int DP>
constexpr int token_waves() {
    return DP * (int)sizeof(T) <= 256 ? 4 : (DP * (int)sizeof(T) <= 512 ? 2 : 1);
}
template <class T, int DP, bool FAST>
__global__ __launch_bounds__(256) void win_token_kernel(TokenArgs a) {
    constexpr int LD = lds_ld<T, DP>(), TILE = WA_BK * LD, NW = token_waves<T, DP>();
    __shared__ __attribute__((aligned(16))) T tiles[NW * TILE];
    __shared__ float sm[NW][16], sl[NW][16], tm[16], tl[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    T* vt = tiles + wave * TILE;
    int id = (int)blockIdx.x;
    const int sp = id % a.splits;
    id /= a.splits;
    const int hg = id % a.hgroups;
    id /= a.hgroups;
    const int hk = id % a.Hkv, b = id / a.Hkv, G = a.Hq / a.Hkv;
    int lo, hi;
    history(a.begin, a.end, b, a.L, lo, hi);
    const int first = hi - a.W > lo ? hi - a.W : lo;                       // window: [first, hi)
    int ns = first - lo < a.S ? first - lo : a.S;                          // first items before it
    if (hi <= lo) ns = 0;
    const int total = hi > lo ? ns + hi - first : 0;
    const int hq = hg * 16 + c16;                                          // query head inside the group
    Oct<T> qf[DP / 32];
    load_frags<T, DP, FAST>(qf, (const T*)a.q + b * a.qb + (hk * G + (hq < G ? hq : 0)) * a.qh, hq < G && total > 0, a.D, a.modeq);
    const T* kp = (const T*)a.k + b * a.ks.b + hk * a.ks.h;
    const T* vp = (const T*)a.v + b * a.vs.b + hk * a.vs.h;
    f32x4 o[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) o[t] = f32x4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.0f;
    const float c = a.scale * WA_LOG2E;
    const int t_end = (sp + 1) * a.per;
    for (int t = sp * a.per + wave; t < t_end && t * WA_BK < total; t += NW) {
        const int n0 = t * WA_BK;
        auto pos = [&](int n) { return (int64_t)(n < ns ? lo + n : first + n - ns); };
        Oct<T> kf[2][DP / 32];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int n = n0 + 16 * y + c16;
            load_frags<T, DP, FAST>(kf[y], kp + pos(n < total ? n : total - 1) * a.ks.l, n < total, a.D, a.mode);
        }
        wave_stage_rows<T, DP, FAST>(vt, vp, a.D, a.mode, [&](int r, bool& ok) {
            ok = n0 + r < total;
            return pos(ok ? n0 + r : total - 1) * a.vs.l;
        });
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) s[y] = mma(kf[y][x], qf[x], s[y]);
        float mt = -__builtin_inff();
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (n0 + 16 * y + 4 * g + i >= total) s[y][i] = -__builtin_inff();
                mt = fmaxf(mt, s[y][i]);
            }
        mt = groups_max(mt);
        const float mn = fmaxf(m, mt), ms = mn == -__builtin_inff() ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f((m - ms) * c);
        m = mn;
        float sum = 0.0f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[y][i] = weight<T>(s[y][i] - ms, c);
                sum += s[y][i];
            }
        l = fmaf(l, alpha, sum);
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) o[x] *= alpha;
        Oct<T> p, pl;                                          // 16-bit types: the halves of P
        if constexpr (sizeof(T) == 2)
            split_oct<T>(s[0], s[1], p, pl);
        else
            p = to_oct<T>(s[0], s[1]);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
            const Oct<T> vf = col_frag<T, LD>(vt, 16 * x);
            o[x] = mma(vf, p, o[x]);
            if constexpr (sizeof(T) == 2) o[x] = mma(vf, pl, o[x]);
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l = groups_sum(l);
    // join the wavefronts: common maximum, then sums in order
    if (g == 0) {
        sm[wave][c16] = m;
        sl[wave][c16] = l;
    }
    __syncthreads();
    float mx = sm[0][c16];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, sm[w][c16]);
    const float ms = mx == -__builtin_inff() ? 0.0f : mx;
    const float f = __builtin_amdgcn_exp2f((m - ms) * c);
    float lt = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) lt += sl[w][c16] * __builtin_amdgcn_exp2f((sm[w][c16] - ms) * c);
    // every wavefront's sums [16 heads][DP] fp32 into its own tile (64 DP bytes of it); one barrier, then they are added
    constexpr int RED = TILE * (int)sizeof(T) / 4;
    float* red = reinterpret_cast<float*>(tiles);
#pragma unroll
    for (int x = 0; x < DP / 16; ++x)
        *reinterpret_cast<f32x4*>(red + wave * RED + c16 * DP + 16 * x + 4 * g) = o[x] * f;
    if (wave == 0 && g == 0) {
        tm[c16] = mx;
        tl[c16] = lt;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * DP; e += NW * 64) {
        const int r = e / DP, d = e % DP, hh = hg * 16 + r;
        if (hh >= G || d >= a.D) continue;
        const int64_t row = (int64_t)b * a.Hq + hk * G + hh;
        const float lr = tl[r];
        float x = red[e];
#pragma unroll
        for (int w = 1; w < NW; ++w) x += red[w * RED + e];
        if (a.splits == 1) {
            ((T*)a.out)[row * a.D + d] = (T)(lr == 0.0f ? 0.0f : x / lr);
        } else {
            float* p = a.part + (row * a.splits + sp) * (a.D + 2);
            p[d] = x;
            if (d == 0) {
                p[a.D] = tm[r];
                p[a.D + 1] = lr;
            }
        }
    }
}
// joins the splits of one query: a thread per split for the common maximum and sum, then 256 / W groups of W lanes take the
// splits in turn (W: D rounded up to 32, 64, .. 256) and are added in order
template <class T>
__global__ __launch_bounds__(256) void win_join_kernel(const float* __restrict__ part, int splits, int D, float scale,
                                                       T* __restrict__ out) {
    __shared__ float f[WA_MAX_SPLITS], red[256], sm[4], sl[4];
    const float* p = part + (int64_t)blockIdx.x * splits * (D + 2);
    const float c = scale * WA_LOG2E;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const bool on = tid < splits;                            // splits <= 256
    const float m = on ? p[(int64_t)tid * (D + 2) + D] : -__builtin_inff(), l = on ? p[(int64_t)tid * (D + 2) + D + 1] : 0.0f;
    float mx = m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if (lane == 0) sm[wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float e = __builtin_amdgcn_exp2f((m - (mx == -__builtin_inff() ? 0.0f : mx)) * c);
    f[tid] = e;
    float lt = l * e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) lt += __shfl_xor(lt, off, 64);
    if (lane == 0) sl[wave] = lt;
    __syncthreads();
    lt = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    const int W = D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256, d = tid % W, groups = 256 / W;
    float o = 0.0f;
    if (d < D)
#pragma unroll 8
        for (int s = tid / W; s < splits; s += groups) o = fmaf(p[(int64_t)s * (D + 2) + d], f[s], o);
    red[tid] = o;
    __syncthreads();
    if (tid >= D) return;
    for (int q = 1; q < groups; ++q) o += red[q * W + tid];
    out[(int64_t)blockIdx.x * D + tid] = (T)(lt == 0.0f ? 0.0f : o / lt);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
// largest of 16, 8, 4, 2 bytes that divides every row start
static int row_alignment(int es, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
    uint64_t bits = 16;
    for (const void* p : bases) bits |= (uint64_t)(uintptr_t)p;
    for (int64_t s : strides) bits |= (uint64_t)(s * es);
    return (int)(bits & (~bits + 1)) > 16 ? 16 : (int)(bits & (~bits + 1));
}
// al: from row_alignment
static int row_mode(int es, int D, int al) {
    if (al >= 16 && D % 8 == 0) return WA_PIECES;
    return es == 4 || (al >= 4 && D % 2 == 0) ? WA_WORDS : WA_ELEMS;
}
// the stride of a dim of one entry is never used and may be anything
static WinStride win_stride(const int64_t* s, int64_t B, int64_t L, int64_t H) {
    return WinStride{B > 1 ? s[0] : 0, L > 1 ? s[1] : 0, H > 1 ? s[2] : 0};
}
static int win_check(const char* who, int64_t B, int64_t L, int32_t Hq, int32_t Hkv, int32_t D, int32_t dtype, int64_t window,
                     int32_t sinks, float scale) {
    DR_REQUIRE(dtype_ok(dtype), "%s: dtype %d", who, dtype);
    DR_REQUIRE(B >= 0 && L >= 1 && L < (1 << 30) && Hq >= 1 && Hkv >= 1 && Hq <= 65536 && Hq % Hkv == 0 && D >= 1 &&
                   D <= WA_MAX_D && B < (1 << 30),
               "%s: bad sizes (B=%lld L=%lld Hq=%d Hkv=%d D=%d)", who, (long long)B, (long long)L, Hq, Hkv, D);
    DR_REQUIRE(window >= 1 && sinks >= 0 && sinks <= WA_MAX_SINKS, "%s: window=%lld (>= 1), sinks=%d (0..%d)", who,
               (long long)window, sinks, WA_MAX_SINKS);
    DR_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "%s: scale must lie in [1e-30, 1e30]", who);
    return DR_OK;
}
template <class Kernel>
static int win_lds(Kernel k, size_t bytes) {
    if (bytes > 65536)
        DR_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return DR_OK;
}
static int64_t win_chunks(int64_t L, int64_t window, int32_t sinks, int group) {
    if (sinks == 0 || L <= window || (L - window + 63) / 64 * group <= 8) return 0;
    return (L + WA_CHUNK - 1) / WA_CHUNK;
}

template <class T, int DP, bool FAST, int NH>
static int win_fwd_heads(const WinArgs& a, void* out, hipStream_t st) {
    const size_t lds = (size_t)fwd_buffers<T, DP>() * 2 * WA_BK * lds_ld<T, DP>() * sizeof(T);
    int rc = win_lds(win_fwd_kernel<T, DP, FAST, NH>, lds);
    if (rc != DR_OK) return rc;
    DR_LAUNCH_NAMED("win_fwd_kernel", (win_fwd_kernel<T, DP, FAST, NH>), dim3((unsigned)a.tiles * (a.Hq / NH) * a.B), dim3(256), lds,
                    st, a, (T*)out, a.lse);
    DR_CHECK_LAUNCH("win_fwd_kernel");
    return DR_OK;
}
template <class T, int DP, bool FAST>
static int win_fwd_launch(const WinArgs& a, void* out, hipStream_t st) {
    // two heads at a time where that leaves 4 workgroups per CU and registers allow: 16 x 2048 x 8 / 2 heads x 64 bf16 58 us
    // against 61, x 32 50 against 52; but x 128 106 against 97, x 64 fp32 209 against 203, and a quarter of the grid 22 against 21
    if constexpr (FAST && DP * (int)sizeof(T) <= 128 && sizeof(T) == 2)
        if (a.Hq / a.Hkv % 2 == 0 && (int64_t)a.tiles * a.Hq * a.B >= 2048) return win_fwd_heads<T, DP, FAST, 2>(a, out, st);
    return win_fwd_heads<T, DP, FAST, 1>(a, out, st);
}
template <class T, int DP, bool FAST>
static int win_bwd_launch(const WinArgs& a, void* dq, void* dk, void* dv, hipStream_t st) {
    const size_t tiles = (size_t)fwd_buffers<T, DP>() * 2 * WA_BK * lds_ld<T, DP>() * sizeof(T);
    const size_t lds = 2 * 64 * lds_ld<T, DP>() * sizeof(T) + 256 * sizeof(float);
    int rc = win_lds(win_dq_kernel<T, DP, FAST>, tiles);
    if (rc != DR_OK) return rc;
    DR_LAUNCH_NAMED("win_dq_kernel", (win_dq_kernel<T, DP, FAST>), dim3((unsigned)a.tiles * a.Hq * a.B), dim3(256), tiles, st, a,
                    (T*)dq);
    DR_CHECK_LAUNCH("win_dq_kernel");
    if (a.chunks > 0) {
        constexpr int NW = sink_waves<T, DP>();
        const size_t sl = (size_t)NW * (2 * WA_BK * lds_ld<T, DP>() * sizeof(T) + 128 * sizeof(float));
        rc = win_lds(win_sink_kernel<T, DP, FAST>, sl);
        if (rc != DR_OK) return rc;
        DR_LAUNCH_NAMED("win_sink_kernel", (win_sink_kernel<T, DP, FAST>), dim3((unsigned)((a.S + 15) / 16) * a.chunks * a.Hkv * a.B),
                        dim3(NW * 64), sl, st, a);
        DR_CHECK_LAUNCH("win_sink_kernel");
    }
    rc = win_lds(win_dkdv_kernel<T, DP, FAST>, lds);
    if (rc != DR_OK) return rc;
    DR_LAUNCH_NAMED("win_dkdv_kernel", (win_dkdv_kernel<T, DP, FAST>), dim3((unsigned)a.ktiles * a.Hkv * a.B), dim3(256), lds, st, a,
                    (T*)dk, (T*)dv);
    DR_CHECK_LAUNCH("win_dkdv_kernel");
    return DR_OK;
}
template <class T, int DP, bool FAST>
static int win_token_launch(const TokenArgs& a, hipStream_t st) {
    DR_LAUNCH_NAMED("win_token_kernel", (win_token_kernel<T, DP, FAST>), dim3((unsigned)a.splits * a.hgroups * a.Hkv * a.B),
                    dim3(64 * token_waves<T, DP>()), 0, st, a);
    DR_CHECK_LAUNCH("win_token_kernel");
    if (a.splits > 1) {
        DR_LAUNCH_NAMED("win_join_kernel", (win_join_kernel<T>), dim3((unsigned)(a.B * a.Hq)), dim3(256), 0, st,
                        (const float*)a.part, a.splits, a.D, a.scale, (T*)a.out);
        DR_CHECK_LAUNCH("win_join_kernel");
    }
    return DR_OK;
}
// workgroups per sequence and key head, 32-key tiles each.  A workgroup's NW wavefronts take NW tiles a round; joining
// costs 3 us, as much as two rounds or more, so up to three rounds stay in one workgroup (64 x 260 keys x 8 / 2 heads x 64
// bf16: 6.5 us so, 8.5 us split in two).  Beyond, the keys are split until there are 2 workgroups per CU or 2 tiles each:
// 1 x 2048 keys takes 7.3 us with 2 tiles each, 8.8 us with 8; 1 x 1000 x 4 heads x 128 fp32 takes 10.9 and 23.4 us.
static void token_split(int64_t B, int Hkv, int hgroups, int64_t keys, int D, int es, int* splits, int* per) {
    const int row = (D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256) * es, nw = row <= 256 ? 4 : (row <= 512 ? 2 : 1);
    const int64_t tiles = (keys + WA_BK - 1) / WA_BK, rows = B * Hkv * hgroups;
    int64_t s = tiles <= 3 * nw ? 1 : (512 + rows - 1) / rows;
    if (s > tiles / 2) s = tiles / 2;
    if (s > WA_MAX_SPLITS) s = WA_MAX_SPLITS;
    if (s < 1) s = 1;
    *per = (int)((tiles + s - 1) / s);
    *splits = (int)((tiles + *per - 1) / *per);
}
static int64_t token_keys(int64_t L, int64_t window, int32_t sinks) { return window >= L ? L : (window + sinks < L ? window + sinks : L); }

// FAST: the head dim fills its tile and rows are read in 16-byte pieces: no column checks anywhere (forward + backward of
// 4 x 2047 x 8 / 2 heads x 128 bf16: 31 + 114 us, 47 + 142 us without; 64 x 200 x 2 x 64 fp32: 18 + 62 and 19 + 66 us)
#define WIN_BY_D(T, fast, launch, ...)                                                                        \
    return a.D <= 32    ? ((fast) && a.D == 32 ? launch<T, 32, true>(__VA_ARGS__) : launch<T, 32, false>(__VA_ARGS__))   \
           : a.D <= 64  ? ((fast) && a.D == 64 ? launch<T, 64, true>(__VA_ARGS__) : launch<T, 64, false>(__VA_ARGS__))   \
           : a.D <= 128 ? ((fast) && a.D == 128 ? launch<T, 128, true>(__VA_ARGS__) : launch<T, 128, false>(__VA_ARGS__)) \
                        : launch<T, 256, false>(__VA_ARGS__)
}  // namespace dr

extern "C" int32_t dr_window_attn_forward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                          const void* v, const int64_t* v_strides, int64_t B, int64_t L, int32_t Hq,
                                          int32_t Hkv, int32_t D, int32_t dtype, int64_t window, int32_t sinks, float scale,
                                          const int32_t* begin, const int32_t* end, void* out, float* lse, void* stream) {
    using namespace dr;
    int rc = win_check("dr_window_attn_forward", B, L, Hq, Hkv, D, dtype, window, sinks, scale);
    if (rc != DR_OK) return rc;
    if (B == 0) return DR_OK;
    DR_REQUIRE(q && k && v && out && lse && q_strides && k_strides && v_strides, "dr_window_attn_forward: NULL pointer");
    const int es = dtype_size(dtype);
    WinArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q;
    a.k = k;
    a.v = v;
    a.qs = win_stride(q_strides, B, L, Hq);
    a.ks = win_stride(k_strides, B, L, Hkv);
    a.vs = win_stride(v_strides, B, L, Hkv);
    a.B = (int)B;
    a.L = (int)L;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    a.W = (int)(window < L ? window : L);
    a.S = sinks;
    a.scale = scale;
    a.begin = begin;
    a.end = end;
    a.lse = lse;
    a.tiles = (int)((L + 63) / 64);
    a.ktiles = (int)((L + 31) / 32);
    DR_REQUIRE((int64_t)a.tiles * Hq * B < WA_MAX_GRID, "dr_window_attn_forward: too many workgroups");
    const int al = row_alignment(es, {q, k, v}, {a.qs.b, a.qs.l, a.qs.h, a.ks.b, a.ks.l, a.ks.h, a.vs.b, a.vs.l, a.vs.h});
    const int alg = row_alignment(es, {out}, {(int64_t)D});
    DR_REQUIRE(al >= es && alg >= es, "dr_window_attn_forward: a pointer is not aligned to its element size");
    a.mode = row_mode(es, D, al);
    a.wide = alg >= 4 * es;
    hipStream_t st = (hipStream_t)stream;
#define WIN_FWD(T) WIN_BY_D(T, a.mode == WA_PIECES && a.wide, win_fwd_launch, a, out, st)
    DR_BY_DTYPE(dtype, WIN_FWD);
#undef WIN_FWD
}

extern "C" int64_t dr_window_attn_backward_bytes(int64_t B, int64_t L, int32_t Hq, int32_t Hkv, int32_t D, int64_t window,
                                                 int32_t sinks) {
    using namespace dr;
    int rc = win_check("dr_window_attn_backward_bytes", B, L, Hq, Hkv, D, DR_F32, window, sinks, 1.0f);
    if (rc != DR_OK) return rc;
    return 3 * align_up(B * Hq * L * 4, 256) + align_up(B * Hq * ((L + 63) / 64) * 16, 256) +
           align_up(B * Hkv * win_chunks(L, window, sinks, Hq / Hkv) * 2 * sinks * D * 4, 256) + 256;
}

extern "C" int32_t dr_window_attn_backward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                           const void* v, const int64_t* v_strides, const void* out, const float* lse,
                                           const void* gout, int64_t B, int64_t L, int32_t Hq, int32_t Hkv, int32_t D,
                                           int32_t dtype, int64_t window, int32_t sinks, float scale, const int32_t* begin,
                                           const int32_t* end, void* dq, void* dk, void* dv, void* ws, int64_t ws_bytes,
                                           void* stream) {
    using namespace dr;
    int rc = win_check("dr_window_attn_backward", B, L, Hq, Hkv, D, dtype, window, sinks, scale);
    if (rc != DR_OK) return rc;
    if (B == 0) return DR_OK;
    DR_REQUIRE(q && k && v && out && lse && gout && dq && dk && dv && q_strides && k_strides && v_strides,
               "dr_window_attn_backward: NULL pointer");
    DR_REQUIRE(ws && aligned_to(ws, 256), "dr_window_attn_backward: workspace is NULL or not 256-byte aligned");
    const int64_t need = dr_window_attn_backward_bytes(B, L, Hq, Hkv, D, window, sinks);
    if (ws_bytes < need)
        DR_FAIL(DR_ERR_WORKSPACE, "dr_window_attn_backward: workspace %lld < required %lld", (long long)ws_bytes, (long long)need);
    const int es = dtype_size(dtype);
    WinArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.gout = gout;
    a.qs = win_stride(q_strides, B, L, Hq);
    a.ks = win_stride(k_strides, B, L, Hkv);
    a.vs = win_stride(v_strides, B, L, Hkv);
    a.B = (int)B;
    a.L = (int)L;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    a.W = (int)(window < L ? window : L);
    a.S = sinks;
    a.scale = scale;
    a.begin = begin;
    a.end = end;
    a.lse = const_cast<float*>(lse);
    a.delta = (float*)ws;
    const int64_t per_query = align_up(B * Hq * L * 4, 256);
    a.ref = (float*)((char*)ws + per_query);
    a.norm = (float*)((char*)ws + 2 * per_query);
    a.gmax = (float*)((char*)ws + 3 * per_query);
    a.part = (float*)((char*)a.gmax + align_up(B * Hq * ((L + 63) / 64) * 16, 256));
    a.chunks = (int)win_chunks(L, window, sinks, Hq / Hkv);
    a.here = sinks > 0 && a.chunks == 0;
    a.tiles = (int)((L + 63) / 64);
    a.ktiles = (int)((L + 31) / 32);
    DR_REQUIRE((int64_t)a.ktiles * Hq * B < WA_MAX_GRID && (int64_t)((sinks + 15) / 16) * a.chunks * Hkv * B < WA_MAX_GRID,
               "dr_window_attn_backward: too many workgroups");
    const int al = row_alignment(es, {q, k, v}, {a.qs.b, a.qs.l, a.qs.h, a.ks.b, a.ks.l, a.ks.h, a.vs.b, a.vs.l, a.vs.h});
    const int alg = row_alignment(es, {out, gout, dq}, {(int64_t)D});
    DR_REQUIRE(al >= es && alg >= es && aligned_to(dk, es) && aligned_to(dv, es),
               "dr_window_attn_backward: a pointer is not aligned to its element size");
    a.mode = row_mode(es, D, al);
    a.modeg = row_mode(es, D, alg);
    a.wide = alg >= 4 * es;
    hipStream_t st = (hipStream_t)stream;
#define WIN_BWD(T) WIN_BY_D(T, a.mode == WA_PIECES && a.modeg == WA_PIECES && a.wide, win_bwd_launch, a, dq, dk, dv, st)
    DR_BY_DTYPE(dtype, WIN_BWD);
#undef WIN_BWD
}

extern "C" int64_t dr_window_attn_token_bytes(int64_t B, int64_t L, int32_t Hq, int32_t Hkv, int32_t D, int64_t window,
                                              int32_t sinks) {
    using namespace dr;
    int rc = win_check("dr_window_attn_token_bytes", B, L, Hq, Hkv, D, DR_F32, window, sinks, 1.0f);
    if (rc != DR_OK) return rc;
    if (B == 0) return 0;
    int splits, more, per;                                     // the types split differently: enough for each
    token_split(B, Hkv, (Hq / Hkv + 15) / 16, token_keys(L, window, sinks), D, 2, &splits, &per);
    token_split(B, Hkv, (Hq / Hkv + 15) / 16, token_keys(L, window, sinks), D, 4, &more, &per);
    if (more > splits) splits = more;
    return splits > 1 ? align_up(B * Hq * splits * ((int64_t)D + 2) * 4, 256) : 0;
}

extern "C" int32_t dr_window_attn_token(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                        const void* v, const int64_t* v_strides, int64_t B, int64_t L, int32_t Hq,
                                        int32_t Hkv, int32_t D, int32_t dtype, int64_t window, int32_t sinks, float scale,
                                        const int32_t* begin, const int32_t* end, void* out, void* ws, int64_t ws_bytes,
                                        void* stream) {
    using namespace dr;
    int rc = win_check("dr_window_attn_token", B, L, Hq, Hkv, D, dtype, window, sinks, scale);
    if (rc != DR_OK) return rc;
    if (B == 0) return DR_OK;
    DR_REQUIRE(q && k && v && out && q_strides && k_strides && v_strides, "dr_window_attn_token: NULL pointer");
    const int64_t need = dr_window_attn_token_bytes(B, L, Hq, Hkv, D, window, sinks);
    DR_REQUIRE(need == 0 || ws != nullptr, "dr_window_attn_token: workspace is NULL");
    DR_REQUIRE(aligned_to(ws, 256), "dr_window_attn_token: workspace is not 256-byte aligned");
    if (ws_bytes < need)
        DR_FAIL(DR_ERR_WORKSPACE, "dr_window_attn_token: workspace %lld < required %lld", (long long)ws_bytes, (long long)need);
    const int es = dtype_size(dtype);
    TokenArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q;
    a.k = k;
    a.v = v;
    a.qb = B > 1 ? q_strides[0] : 0;
    a.qh = Hq > 1 ? q_strides[1] : 0;
    a.ks = win_stride(k_strides, B, L, Hkv);
    a.vs = win_stride(v_strides, B, L, Hkv);
    a.B = (int)B;
    a.L = (int)L;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    a.W = (int)(window < L ? window : L);
    a.S = sinks;
    a.hgroups = (Hq / Hkv + 15) / 16;
    token_split(B, Hkv, a.hgroups, token_keys(L, window, sinks), D, es, &a.splits, &a.per);
    DR_REQUIRE((int64_t)a.splits * a.hgroups * Hkv * B < WA_MAX_GRID && B * Hq < WA_MAX_GRID,
               "dr_window_attn_token: too many workgroups");
    a.scale = scale;
    a.begin = begin;
    a.end = end;
    const int al = row_alignment(es, {k, v}, {a.ks.b, a.ks.l, a.ks.h, a.vs.b, a.vs.l, a.vs.h});
    const int alq = row_alignment(es, {q}, {a.qb, a.qh});
    DR_REQUIRE(al >= es && alq >= es && aligned_to(out, es), "dr_window_attn_token: a pointer is not aligned to its element size");
    a.mode = row_mode(es, D, al);
    a.modeq = row_mode(es, D, alq);
    a.out = out;
    a.part = (float*)ws;
    hipStream_t st = (hipStream_t)stream;
#define WIN_TOK(T) WIN_BY_D(T, a.mode == WA_PIECES && a.modeq == WA_PIECES, win_token_launch, a, st)
    DR_BY_DTYPE(dtype, WIN_TOK);
#undef WIN_TOK
}
