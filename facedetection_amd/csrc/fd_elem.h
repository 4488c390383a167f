// Element types of the expert-block operators: float32, float16 and bfloat16 tensors, arithmetic in float32.
// Rows are read in pieces of 16 bytes from any element-aligned address (gfx950 reads and writes unaligned
// pieces at full width), the last piece of a row element by element.
#pragma once
#include "fd_common.h"

namespace fd {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

inline bool valid_dtype(int t) { return t == FD_F32 || t == FD_F16 || t == FD_BF16; }
inline int dtype_bytes(int t) { return t == FD_F32 ? 4 : 2; }

// runs `f` with a value of the element type as its argument's type
template <typename F>
inline int with_dtype(int t, F&& f) {
    switch (t) {
        case FD_F32: return f(float());
        case FD_F16: return f(_Float16());
        default: return f(__bf16());
    }
}

// P elements from or to p; the one rounding to fewer bits is to nearest even, at the end of an operator
template <int P, typename T>
__device__ __forceinline__ void load_whole(const T* p, float (&v)[P]) {
    T raw[P];
    __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = (float)raw[i];
}
template <int P, typename T>
__device__ __forceinline__ void store_whole(T* p, const float (&v)[P]) {
    T raw[P];
#pragma unroll
    for (int i = 0; i < P; ++i) raw[i] = (T)v[i];
    __builtin_memcpy(p, raw, sizeof(raw));
}

// 8 elements as float32; elements from `n` on are zero and not read, or not written
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if (n >= 8) {
        load_whole<8>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        store_whole<8>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// exp(d) by the hardware's exp2; what d * log2(e) lost in its rounding, and the constant in its own, is put back to first order.
// Off by less than 6 * 2^-24 of the value; a value below 2^-126 is zero.
__device__ __forceinline__ float exp_fast(float d) {
    const float t = d * 1.44269504088896341f, lost = fmaf(d, 1.9259630e-8f, fmaf(d, 1.44269504088896341f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return e > 0.f && e < INFINITY ? fmaf(e, lost * 0.693147180559945309f, e) : e;      // at the ends `lost` is no number
}

// Inclusive scan over a wave, of sums or of the largest value (of values from 0 on): shifts within rows of 16 lanes, then the
// last of row 0 to row 1 and of 2 to 3, then of the half.  Through registers: the six steps by __shfl_up go through LDS, 0.3 us.
template <bool MAX>
__device__ __forceinline__ int wave_scan(int v) {
#define FD_STEP(CTRL, ROWS)                                                             \
    {                                                                                   \
        const int from = __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);     \
        v = MAX ? max(v, from) : v + from;                                              \
    }
    FD_STEP(0x111, 0xf) FD_STEP(0x112, 0xf) FD_STEP(0x114, 0xf) FD_STEP(0x118, 0xf) FD_STEP(0x142, 0xa) FD_STEP(0x143, 0xc)
#undef FD_STEP
    return v;
}

}  // namespace fd
