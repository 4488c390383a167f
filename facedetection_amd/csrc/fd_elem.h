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

// 8 elements from p as float32; elements from `n` on are zero and not read
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if (n >= 8) {
        T raw[8];
        __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}

// the one rounding to fewer bits: to nearest even, at the end of the operator
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        T raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = (T)v[i];
        __builtin_memcpy(p, raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

}  // namespace fd
