// Storage types of the mixed-precision operators (embed, window_attn, logprobs, clip): fp32, fp16 and bf16 elements,
// always widened to fp32 (or fp64) before any arithmetic and rounded once, to nearest even, when stored.
#pragma once
#include "dr_common.h"

namespace dr {

using f16 = _Float16;
using bf16 = __bf16;

template <class T, int V>
struct VecType {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <class T>
struct VecType<T, 1> {
    typedef T type;
};

// V elements at p (aligned to V * sizeof(T)) as floats
template <class T, int V>
__device__ __forceinline__ void load_f32(float (&r)[V], const T* p) {
    if constexpr (V == 1) {
        r[0] = (float)*p;
    } else {
        const typename VecType<T, V>::type t = *reinterpret_cast<const typename VecType<T, V>::type*>(p);
#pragma unroll
        for (int x = 0; x < V; ++x) r[x] = (float)t[x];
    }
}
template <class T, int V>
__device__ __forceinline__ void store_f32(T* p, const float (&r)[V]) {
    if constexpr (V == 1) {
        *p = (T)r[0];
    } else {
        typename VecType<T, V>::type t;
#pragma unroll
        for (int x = 0; x < V; ++x) t[x] = (T)r[x];
        *reinterpret_cast<typename VecType<T, V>::type*>(p) = t;
    }
}

static inline int dtype_size(int dt) { return dt == DR_F32 ? 4 : 2; }
static inline bool dtype_ok(int dt) { return dt == DR_F32 || dt == DR_F16 || dt == DR_BF16; }
static inline bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }

}  // namespace dr

// run `body` (a macro of one type argument) for the element type `dt`
#define DR_BY_DTYPE(dt, body)        \
    do {                             \
        if ((dt) == DR_F32) {        \
            body(float);             \
        } else if ((dt) == DR_F16) { \
            body(dr::f16);           \
        } else {                     \
            body(dr::bf16);          \
        }                            \
    } while (0)
